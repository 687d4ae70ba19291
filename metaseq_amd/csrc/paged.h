// What the kernels of the paged cache share: formats, where positions are, and which rows are whose.
#pragma once

#include "../../include/metaseq_paged.h"
#include "common.h"

// Formats of a page's elements
enum { PG_F16 = 0, PG_BF16 = 1, PG_E4M3 = 2, PG_I8 = 3 };

inline int paged_format(const msa_paged_cache& c) {
  return c.format == MSA_PAGES_E4M3 ? PG_E4M3 : c.format == MSA_PAGES_INT8 ? PG_I8 : c.dtype == MSA_BF16 ? PG_BF16 : PG_F16;
}
inline int paged_log2(int page) { return __builtin_ctz((unsigned)page); }

int msa_paged_check(const msa_paged_cache* c, const msa_paged_batch* b, const char* who);

// Tables name positions below 2^30: one from there on, whichever it is, is nowhere (and a batch's rows behind it are too).
constexpr int PG_NOWHERE = 1 << 30;
// Workgroups of 256 threads that one launch may have (2^32 threads), and rows of a batch.
constexpr int PG_MOST_GROUPS = (1 << 24) - 1;

// attention of a batch, one format of pages (paged_attention_*.hip)
struct PagedAttention {
  const void* q;
  const void *k_pages, *v_pages;
  const int8_t *k_exp, *v_exp;
  const int32_t *seq_start, *seq_pos, *table;
  int64_t ldq, ldo, table_stride;
  void* out;
  // splits > 1: [rows][heads][splits][hd + 4]: sums of p v in units of 2^unit, the maximum m that p is relative to (log2 units), the
  // sum of p, unit (8 bits; 0 with 16), one more for the alignment
  float* partial;
  int M, nseq, heads, kv_heads, pages, page_log2, blocks, out_mb, window, sinks, splits, row_blocks, bf16, max_count;
  int few;      // sequences of at most so many (token, query head) rows of a key/value head are the wave kernel's
  int part_tokens;  // rows of `partial`: so many for each sequence (0: those of the batch)
  int grouped;  // tile kernel: all workgroups of a (sequence, head) on one XCD
  float scale;
};

typedef __attribute__((address_space(4))) int32_t pg_uniform_i32;
typedef uint32_t pg_u2 __attribute__((ext_vector_type(2)));
typedef uint32_t pg_u4 __attribute__((ext_vector_type(4)));

// The sequence of row r: the last one that starts at or before it.  All 64 lanes take part; nseq where r lies in front
// of all (seq_start[0] > r).
__device__ __forceinline__ int paged_sequence_of(const int32_t* __restrict__ seq_start, int nseq, int r) {
  const int lane = threadIdx.x & 63;
  int n = 0;
  for (int base = 0; base < nseq; base += 64) {
    const bool before = base + lane < nseq && seq_start[base + lane] <= r;
    const int c = __popcll(__ballot(before));
    n += c;
    if (c < 64) break;
  }
  return n == 0 ? nseq : n - 1;
}
