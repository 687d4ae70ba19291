/*
 * metaseq_paged.h - the part of libmetaseq_amd.so's C ABI that keeps keys and values in pages: storing new tokens
 * (as they are, or in 8 bits), reading positions back, and attention of new tokens over the pages.
 *
 * Conventions are those of metaseq_amd.h (device pointers, a hipStream_t as `stream`, 0 or a negative msa_status,
 * nothing allocates or synchronises, several threads and devices).  Every pointer to elements is 16-byte aligned and
 * every row stride (in elements) a multiple of 8.
 *
 * The reference appends to one tensor per layer and re-copies its history at every step
 * (metaseq/modules/multihead_attention.py:449-479); pages have no counterpart there.
 */
#ifndef METASEQ_PAGED_H
#define METASEQ_PAGED_H

#include "metaseq_amd.h"

#ifdef __cplusplus
extern "C" {
#endif

enum { MSA_F16 = 2 }; /* beside MSA_BF16 of metaseq_hybrid.h */
enum { MSA_PAGES_SAME = 0, MSA_PAGES_E4M3 = 1, MSA_PAGES_INT8 = 2 };

/* The pages of one layer.  dtype: MSA_F16 or MSA_BF16, the format of k, v, q and out.  format: what the pages hold -
 * MSA_PAGES_SAME: that dtype; MSA_PAGES_E4M3 / _INT8: one byte c per element and one exponent e (int8) per position
 * and head, standing for c 2^e.  k_pages [pages][kv_heads][page][hd], v_pages [pages][kv_heads][hd][page], k_exp and
 * v_exp [pages][kv_heads][page] (NULL with MSA_PAGES_SAME).  page: positions of a page, 16, 32, 64, 128 or 256.
 * hd: 64, 80, 96, 128, 192 or 256. */
typedef struct {
  int dtype, format, kv_heads, hd, page, pages;
  void *k_pages, *v_pages;
  int8_t *k_exp, *v_exp;
} msa_paged_cache;

/* A flat batch: M rows, the new tokens of nseq sequences one behind the other.  seq_start [nseq + 1]: first row of
 * every sequence, and the end of the last one (rows from there on belong to none: nothing is done for them, outputs
 * stay as they were); seq_pos [nseq]: position of its first row (negative: the sequence sits this call out, its
 * outputs stay as they were).  Position p of sequence s is in page table[s * table_stride + p / page]; positions
 * whose entry is outside 0 .. pages - 1, or beyond the `blocks` entries of a sequence, are nowhere: they are not written,
 * read back as zeros and seen by no row.  A table names at
 * most 2^30 positions, a batch has fewer than 2^24 rows.  max_count: no sequence has more rows (those that it has beyond
 * are left alone); min_count: no sequence that has rows has fewer (0: not known); key_bound: no row's position reaches it
 * (a hint: how keys are split follows from it, results up to rounding do not). */
typedef struct {
  int M, nseq, max_count, min_count, key_bound, blocks;
  int64_t table_stride;
  const int32_t *seq_start, *seq_pos, *table;
} msa_paged_batch;

/* Stores keys and values of the batch's rows: k [M, kv_heads, hd] with row stride ldk, v likewise.  8 bits: with top
 * = 448 (e4m3) or 127 (int8), e = the least integer >= -126 with max |x| <= top 2^e over the position's and
 * head's elements, c = x 2^-e rounded to nearest even.  Magnitudes beyond what c 2^e can stand for in dtype (1.875
 * times its largest power of two in e4m3, 1.984375 times it in int8), infinities too, are held as that; NaN is
 * held as e4m3's NaN, in int8 as 0, and is left out of the maximum.  What a position holds that two rows of a call name is
 * undefined (parts of both). */
int msa_paged_append(const msa_paged_cache* c, const msa_paged_batch* b, const void* k, int64_t ldk, const void* v,
                     int64_t ldv, void* stream);

/* Reads the positions of the batch's rows back: k and v [M, kv_heads, hd], c 2^e rounded to dtype. */
int msa_paged_read(const msa_paged_cache* c, const msa_paged_batch* b, void* k, int64_t ldk, void* v, int64_t ldv,
                   void* stream);

/* Attention of the batch's rows over their sequences' pages, which hold the rows' own keys and values already.  Query
 * head h uses key/value head h / (heads / kv_heads).  The row at position i sees positions j <= i, with window > 0 only
 * those of them with j > i - window or j < sinks:
 *   out = sum_j softmax_j(scale q . k_j) v_j
 * with scores, maxima and sums in fp32; probabilities (relative to the maximum) are rounded to 16 bits for their products with
 * values, the result once.  Over 8-bit pages neither a position that a row does not see nor a value that it gives no weight
 * changes its result by more than such a rounding.  A row that sees nothing is zeros.  A row behind its table's positions
 * sees what one at the last of them would.  What stands at positions that no row of a sequence sees is never used, whatever
 * it is.  q [M, heads, hd] with row stride ldq; out with row stride ldo, or (out_mb > 0, MSA_F16, M <= 128) in the packed
 * activation layout of metaseq_amd.h with that many row blocks of heads * hd columns.
 * workspace: at least msa_paged_attention_workspace_bytes of the same arguments (0: none needed), 16-byte aligned; calls
 * that may overlap need one each. */
typedef struct {
  int heads;
  const void* q;
  int64_t ldq;
  void* out;
  int64_t ldo;
  int out_mb, window, sinks;
  float scale;
  void* workspace;
  int64_t workspace_bytes;
} msa_paged_attention_args;
int64_t msa_paged_attention_workspace_bytes(const msa_paged_cache* c, const msa_paged_batch* b,
                                            const msa_paged_attention_args* a);
int msa_paged_attention(const msa_paged_cache* c, const msa_paged_batch* b, const msa_paged_attention_args* a,
                        void* stream);

#ifdef __cplusplus
}
#endif
#endif
