// Storing new tokens' keys and values in pages, as they are or in 8 bits, and reading positions back.
//
// 8 bits: every (position, head) has one exponent e, the least with max |x| <= top 2^e (top = 448 in e4m3, 127 in
// int8), and codes c = x 2^-e rounded to nearest even.  Powers of two make x 2^-e exact, so that a code is the
// only rounding: half a step of e4m3 (2^-4 of the value), which loses nothing by a scale that is not max / 448, or
// half of 2^e in int8 (2^-7 to 2^-8 of the largest, where max / 127 would always be the latter).
#include <math.h>

#include "paged.h"

namespace {

struct PagedRows {
  msa_paged_cache c;
  msa_paged_batch b;
  const void *k, *v;
  void *k_out, *v_out;
  int64_t ldk, ldv;
  int page_log2;
};

template <int DT>
struct Elem;
template <>
struct Elem<MSA_F16> { typedef half_t T; };
template <>
struct Elem<MSA_BF16> { typedef bf16_t T; };

// magnitudes that codes can stand for: see the header
template <int DT, int F>
__device__ __forceinline__ float largest() {
  constexpr float mantissa = F == PG_E4M3 ? 1.875f : 1.984375f;
  return mantissa * (DT == MSA_F16 ? 32768.f : 0x1p127f);
}

// least e >= -126 with amax <= top 2^e (amax >= 0, finite): from the exponent k and the fraction of amax = 1.f 2^k
template <int F>
__device__ __forceinline__ int exponent_of(float amax) {
  const uint32_t w = __builtin_bit_cast(uint32_t, amax);
  const int k = (int)(w >> 23) - 127;
  const uint32_t f = w & 0x7fffff;
  const int e = F == PG_E4M3 ? k - 8 + (f > 0x600000) : k - 6 + (f > 0x7e0000);
  return e < -126 ? -126 : e;
}
// 2^-e (e in -126 .. 120)
__device__ __forceinline__ float inverse_power(int e) { return __builtin_bit_cast(float, (uint32_t)(127 - e) << 23); }

// |x|, and 0 for NaN (the hardware's maximum of a signalling one, as bf16 may hold, is NaN and drops the other operand)
__device__ __forceinline__ float magnitude(float x) { return x != x ? 0.f : fabsf(x); }

// where position p of sequence s is: its page, or -1
__device__ __forceinline__ int page_of(const PagedRows& a, int s, int p) {
  const int block = p >> a.page_log2;
  if (block >= a.b.blocks) return -1;
  const int pg = a.b.table[(int64_t)s * a.b.table_stride + block];
  return pg < 0 || pg >= a.c.pages ? -1 : pg;
}

template <int F>
__device__ __forceinline__ uint32_t code2(float x, float y) {
  if (F == PG_E4M3) return __builtin_amdgcn_cvt_pk_fp8_f32(x, y, 0, false) & 0xffff;
  auto whole = [](float z) { return z != z ? 0u : (uint32_t)(int)rintf(z) & 0xff; };
  return whole(x) | (whole(y) << 8);
}

// One wave per (row, key/value head): the form for few rows per sequence.
template <int DT, int F>
__global__ __launch_bounds__(256) void append_rows_kernel(PagedRows a) {
  typedef typename Elem<DT>::T T;
  const int lane = threadIdx.x & 63, r = blockIdx.x;
  const int h = __builtin_amdgcn_readfirstlane(blockIdx.y * 4 + (threadIdx.x >> 6));
  if (h >= a.c.kv_heads) return;
  const int s = __builtin_amdgcn_readfirstlane(paged_sequence_of(a.b.seq_start, a.b.nseq, r));
  if (s >= a.b.nseq || r >= a.b.seq_start[a.b.nseq] || a.b.seq_pos[s] < 0 || r - a.b.seq_start[s] >= a.b.max_count) return;
  const int p = a.b.seq_pos[s] + r - a.b.seq_start[s];
  const int pg = p < 0 ? -1 : page_of(a, s, p);
  if (pg < 0) return;
  const int hd = a.c.hd, page = 1 << a.page_log2, at = p & (page - 1);
  const int64_t unit = (int64_t)pg * a.c.kv_heads + h;  // of the page and head
  const T* k = (const T*)a.k + (int64_t)r * a.ldk + h * hd;
  const T* v = (const T*)a.v + (int64_t)r * a.ldv + h * hd;
  const int64_t kat = (unit * page + at) * hd, vat = unit * page * hd + at;
  // lane i has elements 2 i, 2 i + 1 and, of heads of more than 128, 128 more
  float kx[4], vx[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int d = (i >> 1) * 128 + 2 * lane + (i & 1);
    kx[i] = d < hd ? (float)k[d] : 0.f;
    vx[i] = d < hd ? (float)v[d] : 0.f;
  }
  if (F < PG_E4M3) {
    T *ko = (T*)a.c.k_pages + kat, *vo = (T*)a.c.v_pages + vat;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int d = (i >> 1) * 128 + 2 * lane + (i & 1);
      if (d < hd) ko[d] = k[d], vo[(int64_t)d * page] = v[d];
    }
    return;
  }
  const float cap = largest<DT, F>();
  float km = 0.f, vm = 0.f;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    km = fmaxf(km, magnitude(kx[i]));
    vm = fmaxf(vm, magnitude(vx[i]));
  }
  const int ke = exponent_of<F>(fminf(wave_max(km), cap)), ve = exponent_of<F>(fminf(wave_max(vm), cap));
  const float ks = inverse_power(ke), vs = inverse_power(ve);
  uint8_t *ko = (uint8_t*)a.c.k_pages + kat, *vo = (uint8_t*)a.c.v_pages + vat;
#pragma unroll
  for (int i = 0; i < 4; i += 2) {
    const int d = (i >> 1) * 128 + 2 * lane;
    if (d >= hd) continue;
    auto held = [&](float x) { return x > cap ? cap : x < -cap ? -cap : x; };
    const uint32_t kc = code2<F>(held(kx[i]) * ks, held(kx[i + 1]) * ks);
    const uint32_t vc = code2<F>(held(vx[i]) * vs, held(vx[i + 1]) * vs);
    *(uint16_t*)(ko + d) = (uint16_t)kc;
    vo[(int64_t)d * page] = (uint8_t)vc;
    vo[(int64_t)(d + 1) * page] = (uint8_t)(vc >> 8);
  }
  if (lane == 0) {
    a.c.k_exp[unit * page + at] = (int8_t)ke;
    a.c.v_exp[unit * page + at] = (int8_t)ve;
  }
}

template <int F>
__device__ __forceinline__ float value_of(uint8_t c) {
  if (F == PG_E4M3) return __builtin_amdgcn_cvt_f32_fp8(c, 0);
  return (float)(int8_t)c;
}

template <int DT, int F>
__global__ __launch_bounds__(256) void read_rows_kernel(PagedRows a) {
  typedef typename Elem<DT>::T T;
  const int lane = threadIdx.x & 63, r = blockIdx.x;
  const int h = __builtin_amdgcn_readfirstlane(blockIdx.y * 4 + (threadIdx.x >> 6));
  if (h >= a.c.kv_heads) return;
  const int s = __builtin_amdgcn_readfirstlane(paged_sequence_of(a.b.seq_start, a.b.nseq, r));
  if (s >= a.b.nseq || r >= a.b.seq_start[a.b.nseq] || a.b.seq_pos[s] < 0 || r - a.b.seq_start[s] >= a.b.max_count) return;
  const int p = a.b.seq_pos[s] + r - a.b.seq_start[s];
  const int pg = p < 0 ? -1 : page_of(a, s, p);
  const int hd = a.c.hd, page = 1 << a.page_log2, at = p & (page - 1);
  T* k = (T*)a.k_out + (int64_t)r * a.ldk + h * hd;
  T* v = (T*)a.v_out + (int64_t)r * a.ldv + h * hd;
  if (pg < 0) {
    for (int d = lane; d < hd; d += 64) k[d] = v[d] = (T)0.f;
    return;
  }
  const int64_t unit = (int64_t)pg * a.c.kv_heads + h, kat = (unit * page + at) * hd, vat = unit * page * hd + at;
  if (F < PG_E4M3) {
    const T *ki = (const T*)a.c.k_pages + kat, *vi = (const T*)a.c.v_pages + vat;
    for (int d = lane; d < hd; d += 64) k[d] = ki[d], v[d] = vi[(int64_t)d * page];
    return;
  }
  const uint8_t *ki = (const uint8_t*)a.c.k_pages + kat, *vi = (const uint8_t*)a.c.v_pages + vat;
  const int ke = a.c.k_exp[unit * page + at], ve = a.c.v_exp[unit * page + at];
  for (int d = lane; d < hd; d += 64) {
    k[d] = (T)ldexpf(value_of<F>(ki[d]), ke);
    v[d] = (T)ldexpf(value_of<F>(vi[(int64_t)d * page]), ve);
  }
}

int check_rows(const msa_paged_cache* c, const msa_paged_batch* b, const void* k, int64_t ldk, const void* v, int64_t ldv,
               const char* who) {
  const int rc = msa_paged_check(c, b, who);
  if (rc) return rc;
  MSA_REQUIRE(k && v, MSA_ERR_INVALID_ARG, "%s: null pointer", who);
  MSA_REQUIRE(((uintptr_t)k | (uintptr_t)v) % 16 == 0, MSA_ERR_INVALID_ARG, "%s: keys and values must be 16-byte aligned", who);
  const int64_t n = (int64_t)c->kv_heads * c->hd;
  MSA_REQUIRE(ldk >= n && ldv >= n && ldk % 8 == 0 && ldv % 8 == 0, MSA_ERR_INVALID_ARG,
              "%s: row strides must be multiples of 8 of at least kv_heads * hd", who);
  return MSA_OK;
}

}  // namespace

int msa_paged_check(const msa_paged_cache* c, const msa_paged_batch* b, const char* who) {
  MSA_REQUIRE(c && b, MSA_ERR_INVALID_ARG, "%s: null pointer", who);
  MSA_REQUIRE(c->dtype == MSA_F16 || c->dtype == MSA_BF16, MSA_ERR_INVALID_ARG, "%s: dtype must be MSA_F16 or MSA_BF16", who);
  MSA_REQUIRE(c->format >= MSA_PAGES_SAME && c->format <= MSA_PAGES_INT8, MSA_ERR_INVALID_ARG, "%s: unknown page format %d", who, c->format);
  MSA_REQUIRE(c->hd == 64 || c->hd == 80 || c->hd == 96 || c->hd == 128 || c->hd == 192 || c->hd == 256, MSA_ERR_INVALID_ARG,
              "%s: head size must be 64, 80, 96, 128, 192 or 256, not %d", who, c->hd);
  MSA_REQUIRE(c->page >= 16 && c->page <= 256 && (c->page & (c->page - 1)) == 0, MSA_ERR_INVALID_ARG,
              "%s: a page must hold 16, 32, 64, 128 or 256 positions, not %d", who, c->page);
  MSA_REQUIRE(c->kv_heads >= 1 && c->kv_heads <= 65535 && c->pages >= 1, MSA_ERR_INVALID_ARG,
              "%s: kv_heads must be 1 .. 65535, pages positive", who);
  MSA_REQUIRE(c->k_pages && c->v_pages, MSA_ERR_INVALID_ARG, "%s: null pointer", who);
  MSA_REQUIRE(c->format == MSA_PAGES_SAME || (c->k_exp && c->v_exp), MSA_ERR_INVALID_ARG, "%s: 8-bit pages need exponents", who);
  MSA_REQUIRE(((uintptr_t)c->k_pages | (uintptr_t)c->v_pages | (uintptr_t)c->k_exp | (uintptr_t)c->v_exp) % 16 == 0,
              MSA_ERR_INVALID_ARG, "%s: pages and exponents must be 16-byte aligned", who);
  MSA_REQUIRE(b->M >= 0 && b->nseq >= 0 && b->nseq <= (1 << 20) && b->max_count >= 0 && b->key_bound >= 0, MSA_ERR_INVALID_ARG,
              "%s: negative sizes, or more than 2^20 sequences", who);
  MSA_REQUIRE(b->blocks >= 1 && b->table_stride >= b->blocks && (int64_t)b->blocks * c->page <= INT32_MAX,
              MSA_ERR_INVALID_ARG, "%s: blocks must be positive, at most table_stride and 2^31 positions", who);
  MSA_REQUIRE(b->nseq == 0 || (b->seq_start && b->seq_pos && b->table), MSA_ERR_INVALID_ARG, "%s: null pointer", who);
  return MSA_OK;
}

#define DISPATCH(kernel)                                                                                     \
  do {                                                                                                       \
    const dim3 grid((unsigned)b->M, (unsigned)((c->kv_heads + 3) / 4));                                      \
    if (c->dtype == MSA_F16) {                                                                               \
      if (c->format == MSA_PAGES_SAME) hipLaunchKernelGGL((kernel<MSA_F16, PG_F16>), grid, dim3(256), 0, s, a);   \
      else if (c->format == MSA_PAGES_E4M3) hipLaunchKernelGGL((kernel<MSA_F16, PG_E4M3>), grid, dim3(256), 0, s, a); \
      else hipLaunchKernelGGL((kernel<MSA_F16, PG_I8>), grid, dim3(256), 0, s, a);                           \
    } else {                                                                                                 \
      if (c->format == MSA_PAGES_SAME) hipLaunchKernelGGL((kernel<MSA_BF16, PG_BF16>), grid, dim3(256), 0, s, a); \
      else if (c->format == MSA_PAGES_E4M3) hipLaunchKernelGGL((kernel<MSA_BF16, PG_E4M3>), grid, dim3(256), 0, s, a); \
      else hipLaunchKernelGGL((kernel<MSA_BF16, PG_I8>), grid, dim3(256), 0, s, a);                          \
    }                                                                                                        \
  } while (0)

extern "C" int msa_paged_append(const msa_paged_cache* c, const msa_paged_batch* b, const void* k, int64_t ldk, const void* v,
                                int64_t ldv, void* stream) {
  const int rc = check_rows(c, b, k, ldk, v, ldv, "msa_paged_append");
  if (rc) return rc;
  if (b->M == 0 || b->nseq == 0 || b->max_count == 0) return MSA_OK;
  hipStream_t s = (hipStream_t)stream;
  const PagedRows a = {*c, *b, k, v, nullptr, nullptr, ldk, ldv, paged_log2(c->page)};
  DISPATCH(append_rows_kernel);
  MSA_CHECK_LAUNCH("msa_paged_append");
  return MSA_OK;
}

extern "C" int msa_paged_read(const msa_paged_cache* c, const msa_paged_batch* b, void* k, int64_t ldk, void* v, int64_t ldv,
                              void* stream) {
  const int rc = check_rows(c, b, k, ldk, v, ldv, "msa_paged_read");
  if (rc) return rc;
  if (b->M == 0 || b->nseq == 0 || b->max_count == 0) return MSA_OK;
  hipStream_t s = (hipStream_t)stream;
  const PagedRows a = {*c, *b, nullptr, nullptr, k, v, ldk, ldv, paged_log2(c->page)};
  DISPATCH(read_rows_kernel);
  MSA_CHECK_LAUNCH("msa_paged_read");
  return MSA_OK;
}
