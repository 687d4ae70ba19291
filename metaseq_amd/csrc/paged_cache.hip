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

// One wave per (row, key/value head): the form for few rows per sequence.  A call of these sizes is latency: where the row belongs,
// its position, its page, then the row.  (Measured: one token of 12 heads of 64 bf16 to e4m3 3.6 us, a plain launch 2 to 3; 32 tokens
// of 32 heads of 128 fp16, whose values are 131072 pieces of two bytes in lines of their own, 7.8 us)
template <int DT, int F>
__global__ __launch_bounds__(256) void append_rows_kernel(PagedRows a) {
  typedef typename Elem<DT>::T T;
  const int lane = threadIdx.x & 63, r = blockIdx.x;
  const int h = __builtin_amdgcn_readfirstlane(blockIdx.y * 4 + (threadIdx.x >> 6));
  if (h >= a.c.kv_heads) return;
  const int s = __builtin_amdgcn_readfirstlane(paged_sequence_of(a.b.seq_start, a.b.nseq, r));
  if (s >= a.b.nseq || r >= a.b.seq_start[a.b.nseq] || a.b.seq_pos[s] < 0 || r - a.b.seq_start[s] >= a.b.max_count) return;
  const int p = min(a.b.seq_pos[s], PG_NOWHERE) + r - a.b.seq_start[s];
  const int pg = page_of(a, s, p);
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

// The other way.  (One token of 12 heads of 64 from e4m3 3.0 us)
template <int DT, int F>
__global__ __launch_bounds__(256) void read_rows_kernel(PagedRows a) {
  typedef typename Elem<DT>::T T;
  const int lane = threadIdx.x & 63, r = blockIdx.x;
  const int h = __builtin_amdgcn_readfirstlane(blockIdx.y * 4 + (threadIdx.x >> 6));
  if (h >= a.c.kv_heads) return;
  const int s = __builtin_amdgcn_readfirstlane(paged_sequence_of(a.b.seq_start, a.b.nseq, r));
  if (s >= a.b.nseq || r >= a.b.seq_start[a.b.nseq] || a.b.seq_pos[s] < 0 || r - a.b.seq_start[s] >= a.b.max_count) return;
  const int p = min(a.b.seq_pos[s], PG_NOWHERE) + r - a.b.seq_start[s];
  const int pg = page_of(a, s, p);
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

// Workgroup = 64 consecutive positions (from a multiple of 64 on) of a sequence, one key/value head: the form for portions of
// prompts.  Rows are read and written 16 bytes a lane; values cross over in LDS, and leave (or come) as 16 bytes of one
// dimension's consecutive positions.  Bound by HBM, 64 positions being a whole line of every dimension in 16 bits.  The heads
// of a block are neighbours, as their pieces of a row are.  (Measured, heads of 128, beside
// a copy's 5.2 TB/s: append of 5047 tokens of 32 heads fp16 to int8, 124 MB, 32 us, 3.9 TB/s, reading them back 22 us, 5.7; of
// 56547 tokens of 8 heads bf16 to e4m3, 348 MB, 82 us, 4.2, and 53 us, 6.6 with part of the pages still cached; reading 25576 tokens
// of 32 heads as they are, 838 MB, 161 us, 5.2.  Appending in 8 bits waits for a row's largest value between loads and stores)
constexpr int PB = 64;  // positions of a block
// From this many new tokens of the longest sequence on the blocks are ahead of a wave for every row, which writes (or reads)
// its values two bytes at a time.  (us, rows and blocks, 64 sequences of 72 heads of 128: fp16 append of 2 15 and 16, of 3 24
// and 18, read of 2 21 and 25, of 3 32 and 26; e4m3 read of 2 12 and 14, of 3 18 and 14, append of 4 26 and 32, of 6 37 and 34;
// a block's 8 bits cross LDS, and 256 sequences of 8 heads append 6 in 19 and 25, 12 in 30 and 29)
constexpr int block_tokens(bool append, int format) { return append && (format == PG_E4M3 || format == PG_I8) ? 6 : 3; }

struct Block {
  int first, begin, end, row;  // positions that are new: begin .. end - 1; the row of position `first`
};
__device__ __forceinline__ bool block_of(const PagedRows& a, int s, int i, Block& b) {
  const pg_uniform_i32* start = (const pg_uniform_i32*)(uintptr_t)a.b.seq_start;
  const int row0 = start[s], pos = min(((const pg_uniform_i32*)(uintptr_t)a.b.seq_pos)[s], PG_NOWHERE);
  const int64_t count = min(min(start[s + 1], a.b.M) - row0, a.b.max_count);
  const int64_t first = ((int64_t)(pos >> 6) + i) * PB;
  if (pos < 0 || row0 < 0 || count <= 0 || first >= pos + count) return false;
  b.first = (int)first;
  b.begin = max(pos, b.first);
  b.end = (int)min(pos + count, first + PB);
  b.row = row0 + b.first - pos;
  return true;
}

// lanes that share a row of HD elements, 8 each: a power of two
template <int HD>
constexpr int row_lanes() { return HD <= 64 ? 8 : HD <= 128 ? 16 : 32; }

// Eight elements of a row that LR lanes share -> their codes and the row's exponent.  The largest magnitude is that of the
// bits; rows that hold a NaN, or more than codes can stand for, take the way of single elements.
template <int DT, int F, int LR>
__device__ __forceinline__ pg_u2 quantise8(pg_u4 w, int& e) {
  typedef typename Elem<DT>::T T;
  typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
  constexpr uint32_t INF = DT == MSA_F16 ? 0x7c00 : 0x7f80;
  auto of = [](uint32_t bits) { return (float)__builtin_bit_cast(T, (uint16_t)bits); };
  auto across = [](float m) {
#pragma unroll
    for (int o = LR / 2; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor(m, o, MSA_WAVE));
    return m;
  };
  u16x2 m2 = {0, 0};
#pragma unroll
  for (int j = 0; j < 4; ++j) m2 = __builtin_elementwise_max(m2, __builtin_bit_cast(u16x2, w[j] & 0x7fff7fffu));
  uint32_t bits = max((uint32_t)m2[0], (uint32_t)m2[1]);
  bits = max(bits, (uint32_t)__builtin_amdgcn_mov_dpp((int)bits, 0xB1, 0xf, 0xf, true));   // the lane next door, the pair
  bits = max(bits, (uint32_t)__builtin_amdgcn_mov_dpp((int)bits, 0x4E, 0xf, 0xf, true));   // next door, the other half of eight
  bits = max(bits, (uint32_t)__builtin_amdgcn_mov_dpp((int)bits, 0x141, 0xf, 0xf, true));  // (mirrored), of sixteen
  if (LR > 8) bits = max(bits, (uint32_t)__builtin_amdgcn_mov_dpp((int)bits, 0x140, 0xf, 0xf, true));
  if (LR > 16) bits = max(bits, (uint32_t)__shfl_xor((int)bits, 16, MSA_WAVE));
  const float cap = largest<DT, F>();
  pg_u2 out;
  if (__ballot(bits > INF || of(bits) > cap)) {
    float x[8], most = 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      x[j] = of(w[j >> 1] >> ((j & 1) * 16));
      most = fmaxf(most, magnitude(x[j]));
    }
    e = exponent_of<F>(fminf(across(most), cap));
    const float f = inverse_power(e);
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = (x[j] > cap ? cap : x[j] < -cap ? -cap : x[j]) * f;
    out[0] = code2<F>(x[0], x[1]) | code2<F>(x[2], x[3]) << 16;
    out[1] = code2<F>(x[4], x[5]) | code2<F>(x[6], x[7]) << 16;
    return out;
  }
  e = exponent_of<F>(of(bits));
  const float f = inverse_power(e);
  if (F == PG_E4M3) {  // (gfx950's conversions from 16 bits with a scale lose the leading bit of subnormals)
    float x[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = of(w[j >> 1] >> ((j & 1) * 16)) * f;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int lo = __builtin_amdgcn_cvt_pk_fp8_f32(x[4 * i], x[4 * i + 1], 0, false);
      out[i] = __builtin_amdgcn_cvt_pk_fp8_f32(x[4 * i + 2], x[4 * i + 3], lo, true);
    }
    return out;
  }
  // int8: the last bits of x 2^-e + 1.5 2^23 are the integer, rounded by the addition (x 2^-e is exact)
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    uint32_t z[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) z[j] = __builtin_bit_cast(uint32_t, __builtin_fmaf(of(w[2 * i + (j >> 1)] >> ((j & 1) * 16)), f, 12582912.f));
    out[i] = __builtin_amdgcn_perm(__builtin_amdgcn_perm(z[3], z[2], 0x0c0c0400u), __builtin_amdgcn_perm(z[1], z[0], 0x0c0c0400u), 0x05040100u);
  }
  return out;
}

// Rows that are read or written once, in whole lines: NT past the caches.
template <bool NT, typename W>
__device__ __forceinline__ W load_once(const void* p) {
  if (NT) return __builtin_nontemporal_load((const W*)p);
  return *(const W*)p;
}
template <bool NT>
__device__ __forceinline__ void store_once(void* p, pg_u4 w) {
  if (NT) __builtin_nontemporal_store(w, (pg_u4*)p);
  else *(pg_u4*)p = w;
}

template <int DT, int F, int HD, bool NT>
__global__ __launch_bounds__(256) void append_block_kernel(PagedRows a, int blocks) {
  typedef typename Elem<DT>::T T;
  constexpr int ES = F < PG_E4M3 ? 2 : 1, LR = row_lanes<HD>(), RP = 256 / LR, N = PB / RP;
  constexpr int STRIDE = HD * ES + 4;                  // of an LDS row: columns are read without bank conflicts
  constexpr int G = 16 / ES, NG = PB / G;              // positions of 16 bytes of a dimension
  __shared__ __attribute__((aligned(16))) char lds[PB * STRIDE];
  // (the heads of a block next to one another: their pieces of a row are)
  const int sb = blockIdx.x / a.c.kv_heads, h = blockIdx.x - sb * a.c.kv_heads, s = sb / blocks;
  const int lane = threadIdx.x % LR, r0 = threadIdx.x / LR;
  Block b;
  if (!block_of(a, s, sb - s * blocks, b)) return;
  const int page = 1 << a.page_log2;
  pg_u4 k[N], v[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int p = b.first + r0 + i * RP;
    k[i] = v[i] = pg_u4{0, 0, 0, 0};
    if (p >= b.begin && p < b.end && lane * 8 < HD) {
      const int64_t row = b.row + r0 + i * RP;
      k[i] = load_once<NT, pg_u4>((const T*)a.k + row * a.ldk + h * HD + lane * 8);
      v[i] = load_once<NT, pg_u4>((const T*)a.v + row * a.ldv + h * HD + lane * 8);
    }
  }
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int p = b.first + r0 + i * RP, at = r0 + i * RP;
    const bool here = p >= b.begin && p < b.end;
    const int pg = here ? page_of(a, s, p) : -1;
    const int64_t unit = (int64_t)pg * a.c.kv_heads + h, place = unit * page + (p & (page - 1));
    if (ES == 2) {
      if (pg >= 0 && lane * 8 < HD) *(pg_u4*)((T*)a.c.k_pages + place * HD + lane * 8) = k[i];
      if (lane * 8 < HD) {
#pragma unroll
        for (int j = 0; j < 4; ++j) *(uint32_t*)(lds + at * STRIDE + lane * 16 + j * 4) = v[i][j];
      }
      continue;
    }
    int ke, ve;
    const pg_u2 kc = quantise8<DT, F, LR>(k[i], ke), vc = quantise8<DT, F, LR>(v[i], ve);
    if (lane * 8 < HD) {
      if (pg >= 0) *(pg_u2*)((uint8_t*)a.c.k_pages + place * HD + lane * 8) = kc;
      *(uint32_t*)(lds + at * STRIDE + lane * 8) = vc[0];
      *(uint32_t*)(lds + at * STRIDE + lane * 8 + 4) = vc[1];
    }
    if (pg >= 0 && lane == 0) a.c.k_exp[place] = (int8_t)ke, a.c.v_exp[place] = (int8_t)ve;
  }
  __syncthreads();
  // a thread turns a word (W dimensions) of G positions into 16 bytes of each dimension
  constexpr int W = 4 / ES;
  for (int i = threadIdx.x; i < HD / W * NG; i += 256) {
    const int d = i / NG * W, g = i % NG, p = b.first + g * G;
    if (p + G <= b.begin || p >= b.end) continue;
    const int pg = page_of(a, s, p);
    if (pg < 0) continue;
    char* to = (char*)a.c.v_pages + ((((int64_t)pg * a.c.kv_heads + h) * HD + d) * page + (p & (page - 1))) * ES;
    const char* from = lds + g * G * STRIDE + d * ES;
    if (p >= b.begin && p + G <= b.end) {
      uint32_t w[G];
      pg_u4 o[W];
#pragma unroll
      for (int j = 0; j < G; ++j) w[j] = *(const uint32_t*)(from + j * STRIDE);
      if (ES == 2) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          o[0][j] = __builtin_amdgcn_perm(w[2 * j + 1], w[2 * j], 0x05040100u);
          o[1][j] = __builtin_amdgcn_perm(w[2 * j + 1], w[2 * j], 0x07060302u);
        }
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint32_t *x = w + 4 * j, lo = __builtin_amdgcn_perm(x[1], x[0], 0x05010400u), hi = __builtin_amdgcn_perm(x[1], x[0], 0x07030602u),
                         lo2 = __builtin_amdgcn_perm(x[3], x[2], 0x05010400u), hi2 = __builtin_amdgcn_perm(x[3], x[2], 0x07030602u);
          o[0][j] = __builtin_amdgcn_perm(lo2, lo, 0x05040100u);
          o[1 % W][j] = __builtin_amdgcn_perm(lo2, lo, 0x07060302u);
          o[2 % W][j] = __builtin_amdgcn_perm(hi2, hi, 0x05040100u);
          o[3 % W][j] = __builtin_amdgcn_perm(hi2, hi, 0x07060302u);
        }
      }
#pragma unroll
      for (int k = 0; k < W; ++k) *(pg_u4*)(to + (int64_t)k * page * ES) = o[k];
    } else {  // positions beside the new ones stay as they are
      for (int j = max(b.begin - p, 0); j < min(b.end - p, G); ++j)
        for (int k = 0; k < W; ++k) {
          if (ES == 2) ((uint16_t*)to)[k * page + j] = *(const uint16_t*)(from + j * STRIDE + k * 2);
          else ((uint8_t*)to)[k * page + j] = *(const uint8_t*)(from + j * STRIDE + k);
        }
    }
  }
}

template <int DT, int F, int HD, bool NT>
__global__ __launch_bounds__(256) void read_block_kernel(PagedRows a, int blocks) {
  typedef typename Elem<DT>::T T;
  constexpr int ES = F < PG_E4M3 ? 2 : 1, LR = row_lanes<HD>(), RP = 256 / LR, N = PB / RP;
  constexpr int STRIDE = HD * ES + 4, G = 16 / ES, NG = PB / G, NV = (HD * NG + 255) / 256;
  __shared__ __attribute__((aligned(16))) char lds[PB * STRIDE];
  // (the heads of a block next to one another: their pieces of a row are)
  const int sb = blockIdx.x / a.c.kv_heads, h = blockIdx.x - sb * a.c.kv_heads, s = sb / blocks;
  const int lane = threadIdx.x % LR, r0 = threadIdx.x / LR;
  Block b;
  if (!block_of(a, s, sb - s * blocks, b)) return;
  const int page = 1 << a.page_log2;
  // 8 codes (or two words more of 16 bits) times 2^e as 16 bytes of T
  auto rows_of = [](pg_u4 w, int e) {
    if (ES == 2) return w;
    pg_u4 out;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t two = w[j >> 1] >> ((j & 1) * 16);
      const T x = (T)ldexpf(value_of<F>((uint8_t)two), e), y = (T)ldexpf(value_of<F>((uint8_t)(two >> 8)), e);
      out[j] = (uint32_t)__builtin_bit_cast(uint16_t, x) | (uint32_t)__builtin_bit_cast(uint16_t, y) << 16;
    }
    return out;
  };
  pg_u4 v[NV], k[N];
  int ke[N], ve[N];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int at = threadIdx.x + i * 256, d = at / NG, p = b.first + (at % NG) * G;
    v[i] = pg_u4{0, 0, 0, 0};
    const int pg = at < HD * NG && p + G > b.begin && p < b.end ? page_of(a, s, p) : -1;
    if (pg >= 0) v[i] = load_once<NT, pg_u4>((const char*)a.c.v_pages + ((((int64_t)pg * a.c.kv_heads + h) * HD + d) * page + (p & (page - 1))) * ES);
  }
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int p = b.first + r0 + i * RP;
    const int pg = p >= b.begin && p < b.end ? page_of(a, s, p) : -1;
    const int64_t place = ((int64_t)pg * a.c.kv_heads + h) * page + (p & (page - 1));
    k[i] = pg_u4{0, 0, 0, 0};
    ke[i] = ve[i] = 0;
    if (pg >= 0 && lane * 8 < HD) {
      if (ES == 2) {
        k[i] = load_once<NT, pg_u4>((const T*)a.c.k_pages + place * HD + lane * 8);
      } else {
        const pg_u2 w = load_once<NT, pg_u2>((const uint8_t*)a.c.k_pages + place * HD + lane * 8);
        k[i][0] = w[0], k[i][1] = w[1];
        ke[i] = a.c.k_exp[place], ve[i] = a.c.v_exp[place];
      }
    }
  }
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int at = threadIdx.x + i * 256;
    if (at >= HD * NG) break;
    char* to = lds + (at % NG) * G * STRIDE + at / NG * ES;
#pragma unroll
    for (int j = 0; j < G; ++j) {
      if (ES == 2) *(uint16_t*)(to + j * STRIDE) = (uint16_t)(v[i][j >> 1] >> ((j & 1) * 16));
      else *(uint8_t*)(to + j * STRIDE) = (uint8_t)(v[i][j >> 2] >> ((j & 3) * 8));
    }
  }
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int p = b.first + r0 + i * RP;
    if (p >= b.begin && p < b.end && lane * 8 < HD)
      store_once<NT>((T*)a.k_out + (int64_t)(b.row + r0 + i * RP) * a.ldk + h * HD + lane * 8, rows_of(k[i], ke[i]));
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int p = b.first + r0 + i * RP;
    if (p < b.begin || p >= b.end || lane * 8 >= HD) continue;
    const char* from = lds + (r0 + i * RP) * STRIDE + lane * 8 * ES;
    pg_u4 w = {0, 0, 0, 0};
#pragma unroll
    for (int j = 0; j < 2 * ES; ++j) w[j] = *(const uint32_t*)(from + j * 4);
    store_once<NT>((T*)a.v_out + (int64_t)(b.row + r0 + i * RP) * a.ldv + h * HD + lane * 8, rows_of(w, ve[i]));
  }
}

template <int DT, int F, int HD>
void launch_rows_hd(const PagedRows& a, bool append, hipStream_t s) {
  if (a.b.max_count < block_tokens(append, F)) {
    const dim3 grid((unsigned)a.b.M, (unsigned)((a.c.kv_heads + 3) / 4));
    if (append) hipLaunchKernelGGL((append_rows_kernel<DT, F>), grid, dim3(256), 0, s, a);
    else hipLaunchKernelGGL((read_rows_kernel<DT, F>), grid, dim3(256), 0, s, a);
    return;
  }
  const int blocks = (a.b.max_count + PB - 2) / PB + 1;  // that max_count positions can meet
  const dim3 grid((unsigned)((int64_t)a.b.nseq * blocks * a.c.kv_heads));
  // Rows of 64 MB and more go past the caches, which the last and the next call could not find them in anyhow (us, through
  // them and past them: read of 8 heads of 128 fp16, 40 MB 14 and 20, 77 MB 38 and 35, 315 MB 134 and 124; of 32 heads from e4m3,
  // 30 MB 12 and 14, 122 MB 46 and 41; append to e4m3, 30 MB 13 and 14, 122 MB 48 and 44; append as they are, 315 MB 140 and 146:
  // never).  Pages are written through the caches: attention reads them next.
  const bool once = (int64_t)a.b.M * a.c.kv_heads * HD * 4 >= 64 << 20;
  if (append) {
    if constexpr (F >= PG_E4M3) {
      if (once) {
        hipLaunchKernelGGL((append_block_kernel<DT, F, HD, true>), grid, dim3(256), 0, s, a, blocks);
        return;
      }
    }
    hipLaunchKernelGGL((append_block_kernel<DT, F, HD, false>), grid, dim3(256), 0, s, a, blocks);
  } else if (once) {
    hipLaunchKernelGGL((read_block_kernel<DT, F, HD, true>), grid, dim3(256), 0, s, a, blocks);
  } else {
    hipLaunchKernelGGL((read_block_kernel<DT, F, HD, false>), grid, dim3(256), 0, s, a, blocks);
  }
}

template <int DT, int F>
void launch_rows_format(const PagedRows& a, bool append, hipStream_t s) {
  switch (a.c.hd) {
    case 64: return launch_rows_hd<DT, F, 64>(a, append, s);
    case 80: return launch_rows_hd<DT, F, 80>(a, append, s);
    case 96: return launch_rows_hd<DT, F, 96>(a, append, s);
    case 128: return launch_rows_hd<DT, F, 128>(a, append, s);
    case 192: return launch_rows_hd<DT, F, 192>(a, append, s);
    default: return launch_rows_hd<DT, F, 256>(a, append, s);
  }
}

void launch_rows(const PagedRows& a, bool append, hipStream_t s) {
  if (a.c.dtype == MSA_F16) {
    if (a.c.format == MSA_PAGES_SAME) return launch_rows_format<MSA_F16, PG_F16>(a, append, s);
    if (a.c.format == MSA_PAGES_E4M3) return launch_rows_format<MSA_F16, PG_E4M3>(a, append, s);
    return launch_rows_format<MSA_F16, PG_I8>(a, append, s);
  }
  if (a.c.format == MSA_PAGES_SAME) return launch_rows_format<MSA_BF16, PG_BF16>(a, append, s);
  if (a.c.format == MSA_PAGES_E4M3) return launch_rows_format<MSA_BF16, PG_E4M3>(a, append, s);
  return launch_rows_format<MSA_BF16, PG_I8>(a, append, s);
}

bool nothing(const msa_paged_batch* b) { return b->M == 0 || b->nseq == 0 || b->max_count == 0; }

int check_rows(const msa_paged_cache* c, const msa_paged_batch* b, const void* k, int64_t ldk, const void* v, int64_t ldv,
               const char* who) {
  const int rc = msa_paged_check(c, b, who);
  if (rc || nothing(b)) return rc;  // (rows that do not exist need no memory)
  MSA_REQUIRE(k && v, MSA_ERR_INVALID_ARG, "%s: null pointer", who);
  MSA_REQUIRE(((uintptr_t)k | (uintptr_t)v) % 16 == 0, MSA_ERR_INVALID_ARG, "%s: keys and values must be 16-byte aligned", who);
  const int64_t n = (int64_t)c->kv_heads * c->hd;
  MSA_REQUIRE((int64_t)b->nseq * (((int64_t)b->max_count + 62) / 64 + 1) * c->kv_heads <= PG_MOST_GROUPS, MSA_ERR_INVALID_ARG, "%s: too many rows for one call", who);
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
  MSA_REQUIRE(b->M <= PG_MOST_GROUPS && b->max_count <= PG_MOST_GROUPS, MSA_ERR_INVALID_ARG, "%s: too many rows for one call", who);
  MSA_REQUIRE(b->M >= 0 && b->nseq >= 0 && b->nseq <= (1 << 20) && b->max_count >= 0 && b->key_bound >= 0, MSA_ERR_INVALID_ARG,
              "%s: negative sizes, or more than 2^20 sequences", who);
  MSA_REQUIRE(b->min_count >= 0 && b->min_count <= b->max_count, MSA_ERR_INVALID_ARG, "%s: min_count must be 0 .. max_count", who);
  MSA_REQUIRE(b->blocks >= 1 && b->table_stride >= b->blocks && (int64_t)b->blocks * c->page <= 1 << 30,
              MSA_ERR_INVALID_ARG, "%s: blocks must be positive, at most table_stride and 2^30 positions", who);
  MSA_REQUIRE(b->nseq == 0 || (b->seq_start && b->seq_pos && b->table), MSA_ERR_INVALID_ARG, "%s: null pointer", who);
  return MSA_OK;
}

extern "C" int msa_paged_append(const msa_paged_cache* c, const msa_paged_batch* b, const void* k, int64_t ldk, const void* v,
                                int64_t ldv, void* stream) {
  const int rc = check_rows(c, b, k, ldk, v, ldv, "msa_paged_append");
  if (rc || nothing(b)) return rc;
  hipStream_t s = (hipStream_t)stream;
  const PagedRows a = {*c, *b, k, v, nullptr, nullptr, ldk, ldv, paged_log2(c->page)};
  launch_rows(a, true, s);
  MSA_CHECK_LAUNCH("msa_paged_append");
  return MSA_OK;
}

extern "C" int msa_paged_read(const msa_paged_cache* c, const msa_paged_batch* b, void* k, int64_t ldk, void* v, int64_t ldv,
                              void* stream) {
  const int rc = check_rows(c, b, k, ldk, v, ldv, "msa_paged_read");
  if (rc || nothing(b)) return rc;
  hipStream_t s = (hipStream_t)stream;
  const PagedRows a = {*c, *b, nullptr, nullptr, k, v, ldk, ldv, paged_log2(c->page)};
  launch_rows(a, false, s);
  MSA_CHECK_LAUNCH("msa_paged_read");
  return MSA_OK;
}
