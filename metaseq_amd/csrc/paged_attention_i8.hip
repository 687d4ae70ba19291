// Attention over pages: int8 pages
#include "paged_attention.h"

void msa_launch_paged_rows_i8(const PagedAttention& a, int hd, int row_tiles, hipStream_t stream) {
  pa_launch_rows_of<PG_I8>(a, hd, row_tiles, stream);
}

bool msa_launch_paged_tiles_i8(const PagedAttention& a, int hd, hipStream_t stream) {
  return pa_launch_tiles_of<PG_I8>(a, hd, stream);
}
