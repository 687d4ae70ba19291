// Attention over pages: bf16 pages
#include "paged_attention.h"

void msa_launch_paged_rows_bf16(const PagedAttention& a, int hd, int row_tiles, hipStream_t stream) {
  pa_launch_rows_of<PG_BF16>(a, hd, row_tiles, stream);
}

bool msa_launch_paged_tiles_bf16(const PagedAttention& a, int hd, hipStream_t stream) {
  return pa_launch_tiles_of<PG_BF16>(a, hd, stream);
}
