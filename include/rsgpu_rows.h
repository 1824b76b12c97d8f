/*
 * rsgpu_rows.h -- rows kept in 8 or 4 bits, the products of a batch's queries with their own partitions' rows, and the rules
 * applied to a batch's scores.  Extensions of the MI355X engine (nothing here exists in VecSim), plain C, pointers and sizes.
 *
 * All arrays below are DEVICE memory and belong to the caller; every call but the two RSGPU_FlatIndex_ ones at the end only launches
 * kernels on `stream` (a hipStream_t; NULL: the device's default stream) and returns: none of them allocates, copies or waits, so they
 * may be captured into a hipGraph.  Two calls that write the same memory are ordered by the caller (one stream, or events).  0 on
 * success, -1 with RSGPU_LastError() otherwise; a refused call has launched nothing.  An index found on the device (a slot, a page,
 * an offset, a list's entry) that is out of its range never leads to an access out of range: what it means is said at each call.
 */
#ifndef RSGPU_ROWS_H
#define RSGPU_ROWS_H

#include <stddef.h>
#include <stdint.h>

#include "VecSim/vec_sim.h"

#ifdef __cplusplus
extern "C" {
#endif

/* ---- a cache of rows ---------------------------------------------------------------------------
 * Row i lives in slot i: RSGPU_RowCache_RowBytes bytes of codes and RSGPU_RowCache_RowScales fp32 scales.  A row is cut into blocks
 * of `block` elements (the last one may be shorter), a block has one scale s, an element x is kept as a code c with x ~ c * s:
 *   INT8    s = (largest |x| of the block) / 127, c = x / s to the nearest integer (ties to even), one signed byte
 *   INT4    the same with 7; two codes a byte, the element of even index in the low four bits, two's complement
 *   E4M3    s = the smallest power of two with |x| <= 448 s, c = x / s as an OCP e4m3 value (nearest, ties to even)
 *   NATIVE  elements as they are (no blocks, no scales; `block` is 0 and `scales` unused)
 * A block whose largest magnitude is below 2^-100 is kept as zeros (s = 0); a block that holds an infinity or a NaN gets s = NaN:
 * it reads back as NaN and so do the products with it.  Elements from dim to the row's end in memory are zeros. */
typedef enum { RSGPU_ROWS_NATIVE = 0, RSGPU_ROWS_INT8 = 1, RSGPU_ROWS_E4M3 = 2, RSGPU_ROWS_INT4 = 3 } RSGPU_RowFormat;

typedef struct RSGPU_RowCache {
  int device;             /* HIP device of the arrays; -1: the one that holds `codes` */
  int type;               /* VecSimType of rows and queries: FLOAT32, FLOAT16 or BFLOAT16 */
  int format;             /* RSGPU_RowFormat */
  uint32_t dim;           /* 1 .. 65536 */
  uint32_t block;         /* elements a scale: 32, 64, 128, or 0: the whole row */
  uint64_t capacity;      /* slots, at most 2^32 - 1 */
  void *codes;            /* capacity * RowBytes, 16-byte aligned */
  float *scales;          /* capacity * RowScales, 4-byte aligned (NULL for NATIVE) */
} RSGPU_RowCache;

/* bytes of one row's codes (dim rounded up to 32 elements), scales of one row; 0: not a cache that is served */
size_t RSGPU_RowCache_RowBytes(const RSGPU_RowCache *cache);
size_t RSGPU_RowCache_RowScales(const RSGPU_RowCache *cache);

/* Row i of `rows` (n rows of dim elements of the cache's type, `stride` elements apart) goes into slot slots[i].  A slot that is
 * negative or not below capacity: the row is left out (padding of a list).  The slots of one call are distinct; of rows that
 * name the same slot, that slot holds any mixture of them, and nothing else is touched.  Other slots are left as they were. */
int RSGPU_RowCache_Write(const RSGPU_RowCache *cache, const void *rows, size_t stride, const int64_t *slots, size_t n, void *stream);

/* rows_out[i] = the row in slot slots[i], each element rounded to the cache's type (one that would
 * pass its largest number is that number); zeros for a slot out of range.  Elements between dim and stride are left as they were.  Slots may come again. */
int RSGPU_RowCache_Read(const RSGPU_RowCache *cache, const int64_t *slots, size_t n, void *rows_out, size_t stride, void *stream);

/* ---- scores of a batch, each query against the rows of its own partition -----------------------
 * Partition g (a tenant, a tag's value) has row_counts[g] rows, row j in slot  pages[g * max_pages + j / page_rows] * page_rows +
 * j % page_rows  of the cache, and the queries query_offsets[g] .. query_offsets[g + 1] - 1 (n_partitions + 1 offsets that do
 * not fall; queries before the first and behind the last belong to nobody).  For each such query m and each j:
 *   scores[m * ld + j] = p  (PRODUCT)  or  1 - p  (DISTANCE: VecSim's inner-product / cosine distance),
 *   p = sum over the elements of query * row, accumulated in fp32 (of rows kept in codes nothing on the way leaves fp32's range
 *   unless such a sum does; bits of an element below 2^-107 and of p below 2^-119 are not kept)
 * A page that is negative or not in the cache: its rows score -inf (PRODUCT) / +inf (DISTANCE), behind every other.  All other
 * cells of `scores` are left as they were.  Right for any groups, fast for even ones: the host chooses the kernel by the queries of a
 * listed partition on average and by max_pages and ld, so list the partitions that are asked.  A row count counts as no more than
 * max_pages * page_rows and ld; a range of queries that falls or leaves [0, n_queries] is cut to it. */
typedef enum { RSGPU_SCORES_PRODUCT = 0, RSGPU_SCORES_DISTANCE = 1 } RSGPU_ScoreForm;

int RSGPU_RowCache_PartitionScores(const RSGPU_RowCache *cache, const void *queries, size_t stride, size_t n_queries,
                                   const int32_t *query_offsets, size_t n_partitions, const int32_t *pages, size_t max_pages,
                                   size_t page_rows, const int32_t *row_counts, int form, float *scores, size_t ld, void *stream);

/* ---- rules on scores: documents already shown, boosts, filters ---------------------------------
 * On the product p of a cell (a DISTANCE score s stands for p = 1 - s), in this order:
 *   shown   the column is n > 0 times in the query's list seen_ids[seen_offsets[m] .. seen_offsets[m + 1] - 1]:
 *           p = p > 0 ? p / repetition[m] : p * repetition[m], then p -= n * frequency[m] + presence[m]
 *   boost   the column is in the query's list bias_ids[..]: p += bias_values[..] (of an id that comes again, the last value)
 *   filter  bit (column % 32) of word column / 32 of the query's mask row is 0: -inf (+inf for a DISTANCE)
 * A cell that no rule touches keeps its bits.  Entries of a list out of [0, n_columns) are passed over; a list's range is cut to
 * [0, n_seen] / [0, n_bias].  (Lists are read once for every 4096 columns: they are meant to be short next to a row of scores.) */
typedef struct RSGPU_ScoreRules {
  int device;                   /* HIP device of the arrays; -1: the one that holds the scores */
  int form;                     /* RSGPU_ScoreForm */
  const uint32_t *mask;         /* n_masks rows of mask_words words; NULL: no filter */
  size_t mask_words, n_masks;
  const int32_t *mask_rows;     /* each query's mask row, one out of [0, n_masks): no filter; NULL: query m has row m */
  const int32_t *bias_offsets;  /* n_queries + 1; NULL: no boosts */
  const int32_t *bias_ids;
  const float *bias_values;
  size_t n_bias;                /* entries of bias_ids and bias_values */
  const int32_t *seen_offsets;  /* n_queries + 1; NULL: nothing shown yet */
  const int32_t *seen_ids;
  size_t n_seen;
  const float *repetition;      /* n_queries each; NULL: 1 */
  const float *frequency;       /* NULL: 0 */
  const float *presence;        /* NULL: 0 */
} RSGPU_ScoreRules;

/* scores_out[m * ld + c] from scores_in[m * ld + c] for c < counts[m] (NULL: n_columns; a count counts as no more than n_columns);
 * other cells of scores_out are left as they were.  scores_out may be scores_in; the two do not overlap otherwise. */
int RSGPU_AdjustScores(const RSGPU_ScoreRules *rules, const float *scores_in, float *scores_out, size_t n_queries, size_t n_columns,
                       size_t ld, const int32_t *counts, void *stream);

/* ---- a FLAT index and a cache ------------------------------------------------------------------
 * The cache has the index's device, dim and type (FLOAT32, FLOAT16, BFLOAT16).  Both calls return when their work is done;
 * `wait_stream` (hipStream_t or NULL) is synchronised first; neither may be captured.  A sharded handle is refused: use its shards. */
/* stored rows [row_begin, row_begin + n) as they are in HBM (cosine rows: normalised) into slots[0 .. n-1], in the order they are
 * stored in: that of their insertion, except that a delete moves the last row into its place.  The cache keeps no labels.  0 or -1. */
int RSGPU_FlatIndex_CacheRows(VecSimIndex *index, size_t row_begin, size_t n, const RSGPU_RowCache *cache, const int64_t *slots,
                              void *wait_stream);
/* n rows of the cache are appended to the index, labelled first_label .. first_label + n - 1, at most 2^64 - 1 (cosine rows are
 * normalised); a slot out of range appends a row of zeros, which a cosine index keeps as every row of zeros, as NaN: behind every
 * other row in its answers.  Returns rows added or -1. */
int RSGPU_FlatIndex_AddCachedRows(VecSimIndex *index, const RSGPU_RowCache *cache, const int64_t *slots, size_t n, size_t first_label,
                                  void *wait_stream);

#ifdef __cplusplus
}
#endif
#endif /* RSGPU_ROWS_H */
