// Attention over pages: which kernel takes a batch, how keys are split, and the sum of the splits.
#include "paged_attention.h"

#define PAGED_FORMAT(name)                                                                      \
  void msa_launch_paged_rows_##name(const PagedAttention& a, int hd, int row_tiles, hipStream_t s); \
  bool msa_launch_paged_tiles_##name(const PagedAttention& a, int hd, hipStream_t s);
PAGED_FORMAT(f16)
PAGED_FORMAT(bf16)
PAGED_FORMAT(e4m3)
PAGED_FORMAT(i8)

namespace {

// out = sum of the splits' sums, each relative to its own maximum.  hd / 4 threads have a (token, query head): a workgroup
// takes several of them, or (MANY) one, for which groups of hd / 4 threads take every so manieth split and their sums are
// added in the groups' order.  tokens: of the sequences of the wave kernel, at most so many each; 0: every row of those of
// the tile kernel (with part_tokens > 0 that many, so that a workgroup's number is its row of the splits' sums).  Bound by its reads, of few rows by latency: 32 splits of 32 heads of 128 of one token 4.7 us.  (us, attention
// and sum, one head to a workgroup and several: 1024 tokens of 32 heads of 128 in 2 splits 74 and 42, in 8 93 and 71, in 16 158
// and 139; 4 tokens in 8 23.7 and 24.2, in 16 21.5 and 23.1, in 32 24 and 28)
constexpr int PC_THREADS = 256, PC_MANY = 9;
template <bool MANY>
__global__ __launch_bounds__(PC_THREADS) void paged_combine_kernel(PagedAttention a, int hd, int tokens) {
  __shared__ __attribute__((aligned(16))) float s_o[MANY ? PC_THREADS : 1][4];
  __shared__ float s_l[MANY ? PC_THREADS : 1];
  const int lane = threadIdx.x & 63, splits = a.splits;
  const bool eight = a.k_exp != nullptr;
  const int s = tokens > 0 ? blockIdx.x / tokens : __builtin_amdgcn_readfirstlane(paged_sequence_of(a.seq_start, a.nseq, blockIdx.x));
  if (s >= a.nseq) return;
  const int row0 = a.seq_start[s], r = tokens > 0 ? row0 + (int)blockIdx.x - s * tokens : (int)blockIdx.x;
  const int count = min(min(a.seq_start[s + 1], a.M) - row0, a.max_count);
  if (a.seq_pos[s] < 0 || row0 < 0 || r - row0 >= count || (count * (a.heads / a.kv_heads) <= a.few) != (tokens > 0)) return;
  const int stride = hd + 4, columns = hd / 4, groups = PC_THREADS / columns;
  const int g = threadIdx.x / columns, c = threadIdx.x - g * columns;
  const int head = MANY ? blockIdx.y : blockIdx.y * groups + g;
  if (!MANY && (g >= groups || head >= a.heads)) return;
  const float* part = a.partial + ((int64_t)(a.part_tokens > 0 ? (int)blockIdx.x : r) * a.heads + head) * splits * stride;
  float top = -INFINITY;
  if constexpr (MANY) {
    for (int i = lane; i < splits; i += 64) top = fmaxf(top, part[i * stride + hd]);
    top = wave_max(top);
  } else {
#pragma unroll 4
    for (int i = 0; i < splits; ++i) top = fmaxf(top, part[i * stride + hd]);
  }
  const float off = top == -INFINITY ? 0.f : top;
  float unit = 0.f;  // of the sum, relative to the maximum
  if (eight) {
    unit = -INFINITY;
    if constexpr (MANY) {
      for (int i = lane; i < splits; i += 64) unit = fmaxf(unit, part[i * stride + hd] - off + part[i * stride + hd + 2]);
      unit = wave_max(unit);
    } else {
#pragma unroll 4
      for (int i = 0; i < splits; ++i) unit = fmaxf(unit, part[i * stride + hd] - off + part[i * stride + hd + 2]);
    }
    unit = unit == -INFINITY ? 0.f : unit;
  }
  float4_t o = {0.f, 0.f, 0.f, 0.f};
  float total = 0.f;
  if (g < groups) {
#pragma unroll 4
    for (int i = MANY ? g : 0; i < splits; i += MANY ? groups : 1) {
      const float4_t v = *(const float4_t*)(part + i * stride + c * 4);
      const float m = part[i * stride + hd] - off, w = __builtin_amdgcn_exp2f(m);
      const float f = eight ? __builtin_amdgcn_exp2f(m + part[i * stride + hd + 2] - unit) : w;
      total += w * part[i * stride + hd + 1];
#pragma unroll
      for (int k = 0; k < 4; ++k) o[k] += f * v[k];
    }
  }
  if constexpr (MANY) {
    *(float4_t*)s_o[threadIdx.x] = o;
    s_l[threadIdx.x] = total;
    __syncthreads();
    if ((int)threadIdx.x >= columns) return;
    for (int i = 1; i < groups; ++i) {
      const float4_t v = *(const float4_t*)s_o[i * columns + c];
      total += s_l[i * columns + c];
#pragma unroll
      for (int k = 0; k < 4; ++k) o[k] += v[k];
    }
  }
  const float inv = total > 0.f || total != total ? 1.f / total : 0.f;
  uint16_t w[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const float x = eight ? pa_times_power(o[k] * inv, unit) : o[k] * inv;
    w[k] = a.bf16 ? __builtin_bit_cast(uint16_t, (bf16_t)x) : __builtin_bit_cast(uint16_t, (half_t)x);
  }
  const int d = head * hd + c * 4;
  const int64_t at = a.out_mb > 0 ? packed_act_offset(r, d, a.out_mb) : (int64_t)r * a.ldo + d;
  *(pg_u2*)((uint16_t*)a.out + at) = pg_u2{(uint32_t)w[0] | (uint32_t)w[1] << 16, (uint32_t)w[2] | (uint32_t)w[3] << 16};
}

// How a batch is taken: sequences of at most few_of() rows (token, query head) of a key/value head by the wave kernel, others
// by tiles; each splits keys over workgroups where there are few of those.  The wave kernel reads the keys once per 32 rows;
// a tile costs the same up to 128, and with 8 bits more, as its operands are made in registers and cross LDS (us, waves and
// tiles, 128 dimensions, 32 query heads: fp16 of as many key/value heads, 16 sequences of 2000 keys, 32 rows 85 and 89, 48
// 116 and 93; 64 sequences of 1000 keys 164 and 183, 211 and 193; 8 heads, 16 sequences 38 and 39, 37 and 40; e4m3, 64 rows
// 98 and 138, 96 rows 138 and 139; 64 sequences 251 and 264, 346 and 281; 8 heads 70 and 75, 97 and 77).
int few_of(const msa_paged_cache& c) { return c.format == MSA_PAGES_SAME ? 32 : 64; }

struct Plan {
  int row_tiles, row_blocks, splits;  // wave kernel (row_tiles 0: not launched)
  int tokens;                         // of a sequence of its, at most
  int64_t tile_blocks;                // tile kernel (0: not launched)
  int tile_splits, grouped;
};

// Splits of the keys, of at least PA_NW tiles each: up to 128 workgroups are made about 256 (one a CU).  Of 129 to 192 some CUs
// would have two and others one: four each share better if they stay long (96 tiles), but for 8 bits of more than 64 dimensions, whose
// workgroups overlap two to a CU.  More are left alone.  (us, attention and sum in 1, 2, 4 splits: 128 workgroups over 700 keys in fp16
// 15, 15, 15, over 4000 68, 49, 50, e4m3 39, 29, 29; 8 over 131072 in int8 80 in 16, 56 in 32, 57 in 64, 60 in 128.  1 and 4 splits:
// fp16, heads of 128, 160 over 2000, 3100, 6200, 16000 keys 40 and 39, 58 and 56, 111 and 103, 275 and 247; 192 42 and 42, 62 and
// 61, 115 and 112, 287 and 273; 224 45 and 51, 67 and 74, 124 and 136, 309 and 332; of 256, 136 72 and 73, 108 and 105, 214 and 194,
// 547 and 472; int8, heads of 64, 156 16 and 18, 24 and 21, 42 and 34, 98 and 74, 240 over 16000 101 and 102; e4m3, heads of 128, 136
// over 6200 and 16000 56 and 56, 127 and 125, 192 59 and 64, 133 and 143, of 256, 136 101 and 109, 236 and 240)
int splits_of(int64_t groups, int64_t tiles, bool overlap) {
  const int64_t most = (tiles + PA_NW - 1) / PA_NW;
  int64_t s = groups <= 128 ? 256 / groups : groups <= 192 && tiles >= 96 && !overlap ? 4 : 1;
  if (s > most) s = most;
  if (s > 128) s = 128;
  return s < 1 ? 1 : (int)s;
}

// The same for tiles: up to one workgroup a CU, of at least 4 tiles each; twice as many, two a CU (where registers and LDS
// allow that, dimensions of up to 128), if each still has more than 16.  (us in 1, 2, 4, 8, 16 splits: 16 workgroups over 4064
// keys 108, 64, 41, 32, 28; 64 over 4064 110, 64, 41, 36, 48; 128 over 8704 227, 131, 102, 115, 150; 256 over 9216 256, 191, 198,
// 231; 256 over 1024 37, 39, 47; of 256 dimensions 32 over 4064 217, 121, 72, 50, 60)
int tile_splits_of(int64_t groups, int64_t tiles, int hd) {
  int64_t s = 256 / groups;
  if (s > tiles / 4) s = tiles / 4;
  if (s < 1) s = 1;
  if (hd <= 128 && groups * s <= 256 && tiles > 16 * s) s *= 2;
  return s > 128 ? 128 : (int)s;
}

Plan plan_of(const msa_paged_cache& c, const msa_paged_batch& b, const msa_paged_attention_args& a) {
  Plan p = {0, 0, 1, 1, 0, 1, 0};
  const int group = a.heads / c.kv_heads;
  const int64_t rows = (int64_t)b.max_count * group;
  // keys that a row block can see
  auto keys_of = [&](int64_t tokens) {
    const int64_t span = (int64_t)a.window + a.sinks + tokens;
    return a.window > 0 && span < b.key_bound ? span : (int64_t)b.key_bound;
  };
  const int few = few_of(c);
  if ((int64_t)b.min_count * group <= few) {
    const int64_t most = rows < few ? rows : few;
    p.row_tiles = most <= 16 ? 1 : 2;
    p.row_blocks = (int)((most + 16 * p.row_tiles - 1) / (16 * p.row_tiles));
    const int kt = c.format == MSA_PAGES_SAME ? 32 : 64;
    const int64_t units = (int64_t)b.nseq * p.row_blocks * c.kv_heads;
    p.splits = splits_of(units, (keys_of(most) + kt - 1) / kt, c.format != MSA_PAGES_SAME && c.hd > 64);
    const int tokens = few / group;
    p.tokens = tokens < 1 ? 1 : tokens < b.max_count ? tokens : b.max_count;
  }
  if (rows > few) {
    p.tile_blocks = (rows + PT_BM - 1) / PT_BM;  // (of as many rows as the caller names: up to 2^40)
    const int64_t units = (int64_t)b.nseq * c.kv_heads;
    p.tile_splits = tile_splits_of(units * p.tile_blocks, (keys_of(PT_BM / group + 1) + PT_BN - 1) / PT_BN, c.hd);
    // A (sequence, head)'s blocks one after another on one XCD, whose L2 then has its keys, where all have about as many:
    // with the long blocks of every unit first the short ones fill the end (us, units first and blocks first: 64 units of 16
    // blocks behind 4096 keys 257 and 301, of 32 behind 1024 204 and 218; 16 units of 128 with a window 178 and 190; from the
    // first key on 32 units of 32 blocks 223 and 178, 256 of 16 314 and 303).  Workgroups go to the XCDs in turn, so that
    // multiples of 8 units keep theirs either way.
    p.grouped = units % 8 == 0 && p.tile_blocks >= 8 && keys_of(b.max_count) >= 2 * (int64_t)(a.window > 0 ? 0 : b.max_count);
  }
  return p;
}

// Rows of the wave kernel's sums in the workspace: where a batch has more than its sequences of that kernel can have (portions
// beside single tokens), so many for each sequence, else the batch's own.
int part_tokens_of(const Plan& p, const msa_paged_batch& b) { return (int64_t)b.nseq * p.tokens < b.M ? p.tokens : 0; }

// The kernels run one after the other and use the same memory.
int64_t partial_floats(const Plan& p, const msa_paged_batch& b, int heads, int hd) {
  const int64_t few = part_tokens_of(p, b) > 0 ? (int64_t)b.nseq * p.tokens : b.M;
  const int64_t rows = p.splits > 1 ? few * p.splits : 0, tiles = p.tile_splits > 1 ? (int64_t)b.M * p.tile_splits : 0;
  return (rows > tiles ? rows : tiles) * heads * (hd + 4);
}

int check(const msa_paged_cache* c, const msa_paged_batch* b, const msa_paged_attention_args* a) {
  const int rc = msa_paged_check(c, b, "msa_paged_attention");
  if (rc) return rc;
  MSA_REQUIRE(a, MSA_ERR_INVALID_ARG, "msa_paged_attention: null pointer");
  MSA_REQUIRE(a->heads >= 1 && a->heads % c->kv_heads == 0, MSA_ERR_INVALID_ARG,
              "msa_paged_attention: %d query heads are no multiple of %d key/value heads", a->heads, c->kv_heads);
  MSA_REQUIRE(a->heads <= 65535, MSA_ERR_INVALID_ARG, "msa_paged_attention: at most 65535 heads");
  MSA_REQUIRE(a->window >= 0 && a->sinks >= 0, MSA_ERR_INVALID_ARG, "msa_paged_attention: window and sinks must not be negative");
  MSA_REQUIRE(a->scale > 0.f && a->scale < INFINITY, MSA_ERR_INVALID_ARG, "msa_paged_attention: scale must be positive and finite");
  return MSA_OK;
}

}  // namespace

extern "C" int64_t msa_paged_attention_workspace_bytes(const msa_paged_cache* c, const msa_paged_batch* b,
                                                       const msa_paged_attention_args* a) {
  const int rc = check(c, b, a);
  if (rc) return rc;
  if (b->M == 0 || b->nseq == 0 || b->max_count == 0) return 0;
  return partial_floats(plan_of(*c, *b, *a), *b, a->heads, c->hd) * 4;
}

extern "C" int msa_paged_attention(const msa_paged_cache* c, const msa_paged_batch* b, const msa_paged_attention_args* a,
                                   void* stream) {
  const int rc = check(c, b, a);
  if (rc) return rc;
  if (b->M == 0 || b->nseq == 0 || b->max_count == 0) return MSA_OK;
  const int64_t width = (int64_t)a->heads * c->hd;
  MSA_REQUIRE(a->q && a->out, MSA_ERR_INVALID_ARG, "msa_paged_attention: null pointer");
  MSA_REQUIRE(((uintptr_t)a->q | (uintptr_t)a->out | (uintptr_t)a->workspace) % 16 == 0, MSA_ERR_INVALID_ARG,
              "msa_paged_attention: queries, outputs and workspace must be 16-byte aligned");
  MSA_REQUIRE(a->ldq >= width && a->ldq % 8 == 0, MSA_ERR_INVALID_ARG, "msa_paged_attention: ldq must be a multiple of 8 of at least heads * hd");
  if (a->out_mb > 0)
    MSA_REQUIRE(c->dtype == MSA_F16 && b->M <= MSA_PACKED_MAX_ROWS && a->out_mb == packed_row_blocks(b->M) && width % 32 == 0,
                MSA_ERR_INVALID_ARG, "msa_paged_attention: packed outputs are fp16, of at most 128 rows and a multiple of 32 columns");
  else
    MSA_REQUIRE(a->out_mb == 0 && a->ldo >= width && a->ldo % 8 == 0, MSA_ERR_INVALID_ARG,
                "msa_paged_attention: ldo must be a multiple of 8 of at least heads * hd");
  const int64_t need = msa_paged_attention_workspace_bytes(c, b, a);
  MSA_REQUIRE(need == 0 || (a->workspace && a->workspace_bytes >= need), MSA_ERR_INVALID_ARG,
              "msa_paged_attention: the workspace has %lld bytes, %lld are needed", (long long)a->workspace_bytes, (long long)need);
  const Plan p = plan_of(*c, *b, *a);
  const int64_t units = (int64_t)b->nseq * c->kv_heads;
  MSA_REQUIRE((int64_t)b->nseq * few_of(*c) <= PG_MOST_GROUPS && units * p.row_blocks <= PG_MOST_GROUPS &&
                  p.tile_blocks <= PG_MOST_GROUPS && (units + 7) * p.tile_blocks * p.tile_splits <= PG_MOST_GROUPS,
              MSA_ERR_INVALID_ARG, "msa_paged_attention: too many rows for one call");
  // (positions are below 2^30; a window that holds them all is none)
  const int window = a->window < (int64_t)b->blocks * c->page ? a->window : 0;
  PagedAttention k = {a->q, c->k_pages, c->v_pages, c->k_exp, c->v_exp, b->seq_start, b->seq_pos, b->table, a->ldq, a->ldo,
                      b->table_stride, a->out, (float*)a->workspace, b->M, b->nseq, a->heads, c->kv_heads, c->pages,
                      paged_log2(c->page), b->blocks, a->out_mb, window, a->sinks, 1, 1,
                      c->dtype == MSA_BF16, b->max_count, few_of(*c), 0, p.grouped, a->scale};
  hipStream_t s = (hipStream_t)stream;
  const int format = paged_format(*c);
  auto combine = [&](int tokens) {
    if (k.splits == 1) return;
    const unsigned x = (unsigned)(tokens > 0 ? b->nseq * tokens : b->M);
    const int each = PC_THREADS / (c->hd / 4);
    if (k.splits >= PC_MANY) hipLaunchKernelGGL(paged_combine_kernel<true>, dim3(x, (unsigned)a->heads), dim3(PC_THREADS), 0, s, k, c->hd, tokens);
    else hipLaunchKernelGGL(paged_combine_kernel<false>, dim3(x, (unsigned)((a->heads + each - 1) / each)), dim3(PC_THREADS), 0, s, k, c->hd, tokens);
  };
  if (p.tile_blocks > 0) {
    k.splits = p.tile_splits;
    k.row_blocks = (int)p.tile_blocks;
    const bool ok = format == PG_F16    ? msa_launch_paged_tiles_f16(k, c->hd, s)
                    : format == PG_BF16 ? msa_launch_paged_tiles_bf16(k, c->hd, s)
                    : format == PG_E4M3 ? msa_launch_paged_tiles_e4m3(k, c->hd, s)
                                        : msa_launch_paged_tiles_i8(k, c->hd, s);
    MSA_REQUIRE(ok, MSA_ERR_HIP, "msa_paged_attention: the kernel's LDS was refused");
    combine(0);
    MSA_CHECK_LAUNCH("msa_paged_attention (tiles)");
  }
  if (p.row_tiles > 0) {
    k.splits = p.splits;
    k.row_blocks = p.row_blocks;
    k.part_tokens = part_tokens_of(p, *b);
    switch (format) {
      case PG_F16: msa_launch_paged_rows_f16(k, c->hd, p.row_tiles, s); break;
      case PG_BF16: msa_launch_paged_rows_bf16(k, c->hd, p.row_tiles, s); break;
      case PG_E4M3: msa_launch_paged_rows_e4m3(k, c->hd, p.row_tiles, s); break;
      default: msa_launch_paged_rows_i8(k, c->hd, p.row_tiles, s); break;
    }
    combine(p.tokens);
    MSA_CHECK_LAUNCH("msa_paged_attention (rows)");
  }
  return MSA_OK;
}
