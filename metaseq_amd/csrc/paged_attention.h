// Attention of few rows per sequence over pages (a decode step, a handful of drafted tokens): the keys are what costs,
// so each is read once for all rows and query heads of its key/value head, and the rows share a wave.
//
// One wave takes KT keys at a time (32 of 16 bits, 64 of 8) and keeps everything in registers; waves share nothing until the end:
//   S^T = K Q^T   v_mfma 16x16x32: a lane has row n = lane % 16 and, of each 16-key tile, four keys
//   O^T += V^T P^T  a lane's probabilities are the B operand as they are, because the key that row m of tile t of S^T
//                 stands for is chosen so: quad q = lane / 16 ends up with KQ consecutive keys q KQ .. + KQ - 1.
// K rows are [position][hd], so 16 bytes of a lane are 8 or 16 dimensions of its key; V is [hd][position], so 16 bytes are
// 8 or 16 consecutive keys of its dimension: the transposed pages spare the product with P every exchange.
//
// Softmax: running maximum m per row, in log2 units, taken over the quads only when a score passes it by more than
// LAZY (probabilities then reach 2^LAZY at most); sums are fp32.  Probabilities are rounded to the 16-bit format that
// the matrix cores take, for fp16 scaled by 2^SHIFT so that they stay normal down to 2^-24 of the maximum.
// 8 bits: a code is exact in fp16.  The key's exponent scales the score; the value's, e, is added to the score, so that what is
// rounded for the product with V is 2^(z - m + e - R), R the row's running maximum of z - m + e: the accumulators are in units of
// 2^(m + R), and neither what other rows see nor a large value without weight takes anything from the row's own.  A second
// exponential for each key hides behind the reads (64 sequences of 72 heads 191 us with it, 191 with one exponent for all
// rows).
//
// Bound by HBM: a key and value cost 4 hd (2 hd) bytes and 4 hd operations a row.  Reads through the caches end at 5.9 to 6.1 TB/s
// here, in pieces of 64 bytes a row or whole lines, in a kernel that does nothing else; whole lines past the caches at 6.7,
// pieces of 64 bytes past them at 6.1, but an operand of the matrix cores is 64 bytes of sixteen rows.  Measured, heads of 128, all
// keys and values: 64 sequences of 1280 keys, 32 heads, fp16, 1.34 GB, 221 us, 6.1 TB/s; 32 of 648 to 1282, 500 MB, 98 us, 5.1
// (and 107 behind an append); 64 sequences, 72 heads, e4m3, 1.07 GB, 191 us, 5.6 TB/s; one of 131072 keys, 8 heads, int8,
// 273 MB, 52 us, 5.3 TB/s, and 5 us for the sum of 32 splits; one of 58 keys, 12 heads of 64, 4.7 us.  Tried without gain: tiles
// of 64 keys of 16 bits (106 us instead of 108), one or two waves a unit, two to four workgroups a CU.
#pragma once

#include <float.h>
#include <math.h>

#include "paged.h"

namespace {

constexpr float PA_LOG2E = 1.4426950408889634f;
constexpr float PA_LAZY = 5.f;
constexpr int PA_NW = 4;  // waves of a workgroup

template <int F>
struct PaFormat {
  static constexpr bool bits8 = F >= PG_E4M3;
  static constexpr int ES = bits8 ? 1 : 2;     // bytes of an element
  static constexpr int KQ = bits8 ? 16 : 8;    // keys of a quad
  static constexpr int KT = 4 * KQ;            // keys of a tile
  static constexpr int NT = KT / 16;           // 16-key tiles of S^T in it
  static constexpr float SHIFT = F == PG_BF16 ? 0.f : 10.f;
};

__device__ __forceinline__ half8_t pa_e4m3(uint32_t lo, uint32_t hi) {
  const half2_t a = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.f, false), b = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.f, true);
  const half2_t c = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.f, false), d = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.f, true);
  return half8_t{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}
// int8 -> fp16: the byte with its sign flipped is the low end of 1024 + c + 128; one subtraction is exact
__device__ __forceinline__ half8_t pa_i8(uint32_t lo, uint32_t hi) {
  lo ^= 0x80808080u;
  hi ^= 0x80808080u;
  const half2_t off = {(half_t)1152.f, (half_t)1152.f};
  auto two = [&](uint32_t w, uint32_t sel) {
    return __builtin_bit_cast(half2_t, __builtin_amdgcn_perm(0x64646464u, w, sel)) - off;
  };
  const half2_t a = two(lo, 0x04010400u), b = two(lo, 0x04030402u), c = two(hi, 0x04010400u), d = two(hi, 0x04030402u);
  return half8_t{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// 16 bytes of a page -> operands of one (16 bits) or two (8 bits) matrix instructions, which are fp16 unless F is bf16
template <int F>
__device__ __forceinline__ pg_u4 pa_operand(pg_u4 w, int half) {
  if (F == PG_E4M3) return __builtin_bit_cast(pg_u4, pa_e4m3(w[2 * half], w[2 * half + 1]));
  if (F == PG_I8) return __builtin_bit_cast(pg_u4, pa_i8(w[2 * half], w[2 * half + 1]));
  return w;
}
template <int F>
__device__ __forceinline__ float4_t pa_mfma(pg_u4 a, pg_u4 b, float4_t c) {
  if (F == PG_BF16)
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8_t, a), __builtin_bit_cast(half8_t, b), c, 0, 0, 0);
}

// Words of values (two of 16 bits, four of 8).  pa_keep: elements whose bit in `seen` is clear become zero.
// pa_not_finite: ones in the places of elements of a kind (1: +infinity, 2: -infinity, 3: NaN; 0: not zero if there is any of
// them).  pa_finite: zeros in their places.
template <int F>
__device__ __forceinline__ uint32_t pa_keep(uint32_t w, uint32_t seen) {
  uint32_t m = 0;
  if (PaFormat<F>::bits8) {
#pragma unroll
    for (int i = 0; i < 4; ++i) m |= seen & (1u << i) ? 0xffu << (8 * i) : 0;
  } else {
    m = (seen & 1 ? 0xffffu : 0) | (seen & 2 ? 0xffff0000u : 0);
  }
  return w & m;
}
template <int F>
__device__ __forceinline__ uint32_t pa_not_finite(uint32_t w, int kind) {
  uint32_t ones = 0;
  if (F == PG_I8) return 0;
  if (F == PG_E4M3) {  // NaN is the one value that is not finite
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (((w >> (8 * i)) & 0x7f) == 0x7f && (kind == 0 || kind == 3)) ones |= 0x38u << (8 * i);
    return ones;
  }
  constexpr uint32_t EXPO = F == PG_BF16 ? 0x7f80u : 0x7c00u, ONE = F == PG_BF16 ? 0x3f80u : 0x3c00u;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const uint32_t x = (w >> (16 * i)) & 0xffff;
    const int is = (x & EXPO) != EXPO ? -1 : (x & (EXPO ^ 0x7fff)) ? 3 : (x & 0x8000) ? 2 : 1;
    if (is == kind || (kind == 0 && is > 0)) ones |= ONE << (16 * i);
  }
  return ones;
}
template <int F>
__device__ __forceinline__ uint32_t pa_finite(uint32_t w) {
  const uint32_t ones = pa_not_finite<F>(w, 0);
  uint32_t out = w;
#pragma unroll
  for (int i = 0; i < (PaFormat<F>::bits8 ? 4 : 2); ++i) {
    const uint32_t m = PaFormat<F>::bits8 ? 0xffu << (8 * i) : 0xffffu << (16 * i);
    if (ones & m) out &= ~m;
  }
  return out;
}

// x 2^e: the power alone may pass what fp32 holds
__device__ __forceinline__ float pa_times_power(float x, float e) {
  const float whole = floorf(e);
  return ldexpf(x * __builtin_amdgcn_exp2f(e - whole), (int)fminf(fmaxf(whole, -1000.f), 1000.f));
}

__device__ __forceinline__ float pa_quads_max(float v) {
  v = fmaxf(v, __shfl_xor(v, 16, MSA_WAVE));
  return fmaxf(v, __shfl_xor(v, 32, MSA_WAVE));
}
__device__ __forceinline__ float pa_quads_sum(float v) {
  v += __shfl_xor(v, 16, MSA_WAVE);
  return v + __shfl_xor(v, 32, MSA_WAVE);
}

// Scores z_j c relative to the maximum m of them, in log2 units, as what exp2 takes is formed in one fused operation: z_j c - off.  The
// maximum is a rounded product, which the fused operation's is not, and far from zero the two differ by more than exp2 can
// take: there (from 2^16 on in some lane) z becomes the rounded products less the maximum, c one.  m = -infinity: no score yet.
constexpr float PA_FAR = 65536.f;
template <int N>
__device__ __forceinline__ void pa_relative(float (&z)[N], float& c, float& off, float m, float shift) {
#pragma clang fp contract(off)
  const float from = m == -INFINITY ? 0.f : m;
  off = from - shift;
  if (__builtin_expect(__ballot(fabsf(from) >= PA_FAR) != 0, 0)) {
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const float score = z[j] * c;
      z[j] = score - from;
    }
    c = 1.f;
    off = -shift;
  }
}

// Of the N keys from `key` on (N <= 16), as bits, those that some row at a position between lo and hi sees (of
// consecutive tokens; lo == hi: that the row sees).
template <int N>
__device__ __forceinline__ uint32_t pa_seen(int key, int lo, int hi, int window, int sinks) {
  auto upto = [&](int last) { return (1u << min(max(last - key + 1, 0), N)) - 1; };  // keys <= last
  const uint32_t past = upto(hi);
  return window > 0 ? past & (~upto(lo - window) | upto(sinks - 1)) : past;
}

// The tiles of KT keys that rows at positions lo .. hi see: those of the first `sinks` positions, then from the window's
// start on.
template <int KT>
struct PaTiles {
  int head, first, n;  // tiles of the first positions; first tile behind them; all
  __device__ __forceinline__ PaTiles(int lo, int hi, int window, int sinks) {
    const int w0 = window > 0 && window <= lo ? lo - window + 1 : 0;  // (window <= lo: no overflow)
    first = w0 / KT;
    head = min((min(sinks, hi + 1) + KT - 1) / KT, first);
    n = head + hi / KT - first + 1;
  }
  __device__ __forceinline__ int tile(int i) const { return i < head ? i : first + i - head; }
};

// pages of a tile's four groups of sixteen keys, -1: none
struct PtPages {
  int a, b, c, d;
  __device__ __forceinline__ int of(int g16) const {
    const int w = a, x = b, y = c, z = d;
    return g16 < 2 ? (g16 < 1 ? w : x) : (g16 < 3 ? y : z);
  }
};

template <int F, int HD, int RT>
__global__ __launch_bounds__(PA_NW * 64) void paged_rows_kernel(PagedAttention a) {
  typedef PaFormat<F> X;
  constexpr bool B8 = X::bits8;
  constexpr int ES = X::ES, KQ = X::KQ, KT = X::KT, NT = X::NT;
  constexpr int CD = 16 / ES * 4;              // dimensions that one load instruction covers: 32 or 64
  constexpr int KL = (HD + CD - 1) / CD;       // load instructions of a 16-key tile
  constexpr int HALVES = B8 ? 2 : 1;           // matrix instructions to a load
  constexpr int DT = HD / 16;                  // 16-dimension tiles of O^T
  constexpr int LDO = HD + 4;
  __shared__ __attribute__((aligned(16))) float s_acc[PA_NW][16][LDO];
  static_assert(16 * LDO * 4 >= HD * KT * ES, "a tile's values of one wave");
  __shared__ float s_m[PA_NW][16], s_l[PA_NW][16], s_r[B8 ? PA_NW : 1][16];

  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n16 = lane & 15, quad = lane >> 4;
  // (the heads of a sequence next to one another, as they are in its pages)
  const int srb = blockIdx.x / a.kv_heads, h = blockIdx.x - srb * a.kv_heads, split = blockIdx.y;
  const int s = srb / a.row_blocks, rb = srb - s * a.row_blocks;
  const int group = a.heads / a.kv_heads;
  const pg_uniform_i32* seq_start = (const pg_uniform_i32*)(uintptr_t)a.seq_start;
  const int row0 = seq_start[s], pos = ((const pg_uniform_i32*)(uintptr_t)a.seq_pos)[s];
  const int count = min(min(seq_start[s + 1], a.M) - row0, a.max_count);
  if (pos < 0 || row0 < 0 || count <= 0 || count * group > a.few || rb * 16 * RT >= count * group) return;
  const int page = 1 << a.page_log2, rows = count * group, rho0 = rb * 16 * RT;
  const int limit = a.blocks * page - 1;  // last position that can be anywhere
  const int p_lo = (int)min((int64_t)pos + rho0 / group, (int64_t)limit);
  const int p_hi = (int)min((int64_t)pos + (min(rho0 + 16 * RT, rows) - 1) / group, (int64_t)limit);
  const PaTiles<KT> tiles(p_lo, p_hi, a.window, a.sinks);
  // this split's tiles, every PA_NW-th of them this wave's
  const int per = (tiles.n + a.splits - 1) / a.splits, it_end = min(tiles.n, (split + 1) * per);

  // ---- queries: B operand, row n16 of row tile rt, the dimensions that the lane's loads of K have ----
  pg_u4 qf[RT][KL][HALVES];
  const float qs = a.scale * PA_LOG2E;  // what turns a product into a score in log2 units
  int eq[RT];    // 8 bits: the power of two that the row's queries stand for
  int pn[RT];    // the row's position; rows past the last one see nothing
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    const int rho = rho0 + rt * 16 + n16;
    const bool live = rho < rows;
    const int t = live ? rho / group : 0, g = live ? rho - t * group : 0;
    pn[rt] = live ? (int)min((int64_t)pos + t, (int64_t)limit) : -1;
    const char* q = (const char*)a.q + (((int64_t)row0 + t) * a.ldq + (int64_t)(h * group + g) * HD) * 2;
    eq[rt] = 0;
#pragma unroll
    for (int c = 0; c < KL; ++c)
#pragma unroll
      for (int e = 0; e < HALVES; ++e) {
        const int d = c * CD + quad * (CD / 4) + e * 8;
        qf[rt][c][e] = d < HD ? *(const pg_u4*)(q + d * 2) : pg_u4{0, 0, 0, 0};
      }
    if (B8 && a.bf16) {  // to fp16: the row times a power of two that brings its largest to 2^8
      float big = 0.f;
#pragma unroll
      for (int c = 0; c < KL; ++c)
#pragma unroll
        for (int e = 0; e < HALVES; ++e) {
          const bf16x8_t v = __builtin_bit_cast(bf16x8_t, qf[rt][c][e]);
#pragma unroll
          for (int i = 0; i < 8; ++i) big = fmaxf(big, fabsf((float)v[i]));
        }
      big = pa_quads_max(big);
      const int k = min(max((int)(__builtin_bit_cast(uint32_t, big) >> 23) - 127 - 8, -118), 120);
#pragma unroll
      for (int c = 0; c < KL; ++c)
#pragma unroll
        for (int e = 0; e < HALVES; ++e) {
          const bf16x8_t v = __builtin_bit_cast(bf16x8_t, qf[rt][c][e]);
          half8_t w;
#pragma unroll
          for (int i = 0; i < 8; ++i) w[i] = (half_t)ldexpf((float)v[i], -k);
          qf[rt][c][e] = __builtin_bit_cast(pg_u4, w);
        }
      eq[rt] = k;
    }
  }

  float4_t acc[RT][DT];
  float m[RT], l[RT], R[RT];
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    m[rt] = R[rt] = -INFINITY;
    l[rt] = 0.f;
#pragma unroll
    for (int d = 0; d < DT; ++d) acc[rt][d] = float4_t{0.f, 0.f, 0.f, 0.f};
  }

  // ---- tiles.  As a source of K a lane has keys of quad n16 / 4, as one of V of its own quad.  Keys and values are
  // requested a tile ahead, each into the registers that the matrix instructions have just read.  (Nothing past the caches: a
  // line of keys is two instructions', one of values two tiles'.  32 sequences of 32 heads over 640 to 1281 keys in fp16, us:
  // 135 with everything past them, 107 so) ----
  const pg_uniform_i32* table = (const pg_uniform_i32*)(uintptr_t)(a.table + (int64_t)s * a.table_stride);
  // page of the sixteen keys g16 of tile i, -1 where there is none
  auto look = [&](int i, int g16) {
    const int block = (tiles.tile(i) * KT + g16 * 16) >> a.page_log2;
    const int pg = table[min(block, a.blocks - 1)];
    return block < a.blocks && (unsigned)pg < (unsigned)a.pages ? pg : -1;
  };
  auto look4 = [&](int i) {
    i = min(i, it_end - 1);
    return PtPages{look(i, 0), look(i, 1), B8 ? look(i, 2) : 0, B8 ? look(i, 3) : 0};
  };
  auto of_quad = [](PtPages pg, int q) { return B8 ? pg.of(q) : pg.of(q >> 1); };
  const int64_t unit = (int64_t)page * HD * ES;  // bytes of a page and head
  pg_u4 kf[NT][KL], vf[DT];
  auto load_k = [&](int i, PtPages pages) {
    const int key = tiles.tile(i) * KT + (n16 >> 2) * KQ + (n16 & 3), pg = of_quad(pages, n16 >> 2);
    const char* base = (const char*)a.k_pages + ((int64_t)max(pg, 0) * a.kv_heads + h) * unit + (int64_t)(key & (page - 1)) * (HD * ES) + quad * 16;
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int c = 0; c < KL; ++c)
        kf[t][c] = (c + 1) * CD <= HD || quad * (CD / 4) + c * CD < HD
                       ? *(const pg_u4*)(base + t * 4 * HD * ES + c * 64)
                       : pg_u4{0, 0, 0, 0};
  };
  auto load_v = [&](int i, PtPages pages) {
    const int key = tiles.tile(i) * KT + quad * KQ, pg = of_quad(pages, quad);
    const char* base = (const char*)a.v_pages + ((int64_t)max(pg, 0) * a.kv_heads + h) * unit + (n16 * page + (key & (page - 1))) * ES;
#pragma unroll
    for (int d = 0; d < DT; ++d) vf[d] = *(const pg_u4*)(base + d * 16 * page * ES);
  };
  pg_u4 kx, vx;  // exponents of the quad's keys
  auto load_x = [&](int i, PtPages pages) {
    const int key = tiles.tile(i) * KT + quad * KQ, pg = of_quad(pages, quad);
    const int64_t at = ((int64_t)max(pg, 0) * a.kv_heads + h) * page + (key & (page - 1));
    kx = *(const pg_u4*)(a.k_exp + at);
    vx = *(const pg_u4*)(a.v_exp + at);
  };
  auto byte_of = [](pg_u4 w, int i) { return (int)(int8_t)(w[i >> 2] >> ((i & 3) * 8)); };

  int i = split * per + wave;
  PtPages pg = {-1, -1, -1, -1}, next = pg;  // of this tile and the wave's next one
  if (i < it_end) {
    pg = look4(i);
    next = look4(i + PA_NW);
    load_k(i, pg);
    if (B8) load_x(i, pg);
    load_v(i, pg);
  }
  // MORE: there is a next tile of this wave's.  (The last one has a copy of its own: behind a branch around the requests
  // every wait would be for all of them.)
  auto step = [&](auto more) {
    constexpr bool MORE = decltype(more)::value;
    const int key0 = tiles.tile(i) * KT;  // of the tile
    const int kq = key0 + quad * KQ;      // of the quad
    const bool there = of_quad(pg, quad) >= 0;
    // every row sees every key of the tile
    const bool whole = key0 + KT - 1 <= p_lo && (a.window <= 0 || key0 > p_hi - a.window || key0 + KT <= a.sinks) &&
                       (pg.a | pg.b | pg.c | pg.d) >= 0;
    // the quad's keys that some row sees
    const uint32_t seen = whole ? ~0u : there ? pa_seen<KQ>(kq, p_lo, p_hi, a.window, a.sinks) : 0;
    float z[RT][KQ];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      float4_t sc[RT];
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) sc[rt] = float4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int c = 0; c < KL; ++c)
#pragma unroll
        for (int e = 0; e < HALVES; ++e) {
          const pg_u4 k = pa_operand<F>(kf[t][c], e);
#pragma unroll
          for (int rt = 0; rt < RT; ++rt) sc[rt] = pa_mfma<F>(k, qf[rt][c][e], sc[rt]);
        }
#pragma unroll
      for (int rt = 0; rt < RT; ++rt)
#pragma unroll
        for (int e = 0; e < 4; ++e) z[rt][t * 4 + e] = sc[rt][e];
    }
    if (MORE) load_k(i + PA_NW, next);
    pg_u4 pf[RT][HALVES];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      const uint32_t sees = there ? pa_seen<KQ>(kq, pn[rt], pn[rt], a.window, a.sinks) : 0;
      float top = -INFINITY;
#pragma unroll
      for (int j = 0; j < KQ; ++j) {
        if (B8) z[rt][j] = ldexpf(z[rt][j], byte_of(kx, j) + eq[rt]);  // (either alone may pass what fp32 holds)
        z[rt][j] = (sees >> j) & 1 ? z[rt][j] : -INFINITY;
        top = fmaxf(top, z[rt][j]);
      }
      top *= qs;
      if (__ballot(top > m[rt] + PA_LAZY)) {  // (m = -inf: any score)
        const float to = fmaxf(m[rt], pa_quads_max(top));
        const float w = m[rt] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m[rt] - to);
        if (B8) {
          R[rt] -= m[rt] == -INFINITY ? 0.f : to - m[rt];
        } else {
#pragma unroll
          for (int d = 0; d < DT; ++d)
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[rt][d][e] *= w;
        }
        m[rt] = to;
        l[rt] *= w;
      }
      float c = qs, off;
      pa_relative(z[rt], c, off, m[rt], B8 ? 0.f : X::SHIFT);
      float p[KQ], sum = 0.f;
#pragma unroll
      for (int j = 0; j < KQ; ++j) {
        z[rt][j] = __builtin_fmaf(z[rt][j], c, -off);
        p[j] = __builtin_amdgcn_exp2f(z[rt][j]);
        sum += p[j];
      }
      l[rt] += sum;
      if (B8) {
        float most = -INFINITY;
#pragma unroll
        for (int j = 0; j < KQ; ++j) {
          z[rt][j] += (float)byte_of(vx, j);
          most = fmaxf(most, z[rt][j]);
        }
        if (__ballot(most > R[rt] + PA_LAZY)) {
          const float to = fmaxf(R[rt], pa_quads_max(most)), w = R[rt] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(R[rt] - to);
          R[rt] = to;
#pragma unroll
          for (int d = 0; d < DT; ++d)
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[rt][d][e] *= w;
        }
        const float from = (R[rt] == -INFINITY ? 0.f : R[rt]) - X::SHIFT;
#pragma unroll
        for (int j = 0; j < KQ; ++j) p[j] = __builtin_amdgcn_exp2f(z[rt][j] - from);
      }
#pragma unroll
      for (int e = 0; e < HALVES; ++e) {
        if (F == PG_BF16) {
          bf16x8_t w;
#pragma unroll
          for (int j = 0; j < 8; ++j) w[j] = (bf16_t)p[e * 8 + j];
          pf[rt][e] = __builtin_bit_cast(pg_u4, w);
        } else {
          half8_t w;
#pragma unroll
          for (int j = 0; j < 8; ++j) w[j] = (half_t)p[e * 8 + j];
          pf[rt][e] = __builtin_bit_cast(pg_u4, w);
        }
      }
    }
    if (B8 && MORE) load_x(i + PA_NW, next);
    if (!whole) {
      // Keys that no row sees may hold anything: their values are taken as zeros.  A value that is not finite at a key
      // that some rows see and others do not must reach those rows only (0 times infinity is NaN): it is added to those
      // and left out of the product.
      pg_u4 keep;
#pragma unroll
      for (int k = 0; k < 4; ++k) keep[k] = pa_keep<F>(~0u, seen >> (k * (KQ / 4)));
      bool odd = false;
#pragma unroll
      for (int d = 0; d < DT; ++d) {
        vf[d] &= keep;
#pragma unroll
        for (int k = 0; k < 4; ++k) odd |= pa_not_finite<F>(vf[d][k], 0) != 0;
      }
      if (F != PG_I8 && __ballot(odd)) {  // (an infinity or a NaN times a probability is itself)
        char* vt = (char*)s_acc[wave];    // [dimension][key]; not used before the end
#pragma unroll
        for (int d = 0; d < DT; ++d) *(pg_u4*)(vt + ((d * 16 + n16) * KT + quad * KQ) * ES) = vf[d];
#pragma unroll 1
        for (int j = 0; j < KT; ++j) {
          const char* at = vt + (quad * 4 * KT + j) * ES;
          const bool anywhere = of_quad(pg, j / KQ) >= 0;
          bool mine[RT];
#pragma unroll
          for (int rt = 0; rt < RT; ++rt) mine[rt] = anywhere && pa_seen<1>(key0 + j, pn[rt], pn[rt], a.window, a.sinks);
#pragma unroll
          for (int d = 0; d < DT; ++d)
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const char* x = at + (d * 16 + k) * KT * ES;
              const float f = B8 ? ((*(const uint8_t*)x & 0x7f) == 0x7f ? NAN : 0.f)
                                 : F == PG_BF16 ? (float)*(const bf16_t*)x : (float)*(const half_t*)x;
#pragma unroll
              for (int rt = 0; rt < RT; ++rt) acc[rt][d][k] += (mine[rt] & !(fabsf(f) < INFINITY)) ? f : 0.f;
            }
        }
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
          for (int k = 0; k < 4; ++k) vf[d][k] = pa_finite<F>(vf[d][k]);
      }
    }
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
      for (int e = 0; e < HALVES; ++e) {
        const pg_u4 v = pa_operand<F>(vf[d], e);
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) acc[rt][d] = pa_mfma<F>(v, pf[rt][e], acc[rt][d]);
      }
    if (MORE) load_v(i + PA_NW, next);
  };
#pragma unroll 1
  for (; i + PA_NW < it_end; i += PA_NW) {
    step(std::true_type{});
    pg = next;
    next = look4(i + 2 * PA_NW);
  }
  if (i < it_end) step(std::false_type{});

  // ---- the waves' sums: one row tile at a time through LDS, added in the waves' order ----
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    const int left = min(16, rows - rho0 - rt * 16);
    if (left <= 0) break;
    l[rt] = pa_quads_sum(l[rt]);
    if (rt > 0) __syncthreads();
    if (quad == 0) {
      s_m[wave][n16] = m[rt], s_l[wave][n16] = l[rt];
      if (B8) s_r[wave][n16] = R[rt] - X::SHIFT;
    }
    if (n16 < left) {
#pragma unroll
      for (int d = 0; d < DT; ++d) *(float4_t*)&s_acc[wave][n16][d * 16 + quad * 4] = acc[rt][d];
    }
    __syncthreads();
    for (int j = threadIdx.x; j < left * (HD / 4); j += PA_NW * 64) {
      const int r = j / (HD / 4), d = (j - r * (HD / 4)) * 4;
      float to = -INFINITY;
#pragma unroll
      for (int w = 0; w < PA_NW; ++w) to = fmaxf(to, s_m[w][r]);
      const float off = to == -INFINITY ? 0.f : to;
      float total = 0.f, unit = 0.f;  // (8 bits: o is in units of 2^unit)
      if (B8) {
        unit = -INFINITY;
#pragma unroll
        for (int w = 0; w < PA_NW; ++w) unit = fmaxf(unit, s_m[w][r] - off + s_r[w][r]);
        unit = unit == -INFINITY ? 0.f : unit;
      }
      float4_t o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int w = 0; w < PA_NW; ++w) {
        const float f = __builtin_amdgcn_exp2f(s_m[w][r] - off), g = B8 ? __builtin_amdgcn_exp2f(s_m[w][r] - off + s_r[w][r] - unit) : f;
        total += f * s_l[w][r];
        const float4_t v = *(const float4_t*)&s_acc[w][r][d];
#pragma unroll
        for (int k = 0; k < 4; ++k) o[k] += g * v[k];
      }
      const int rho = rho0 + rt * 16 + r, t = rho / group, head = h * group + rho - t * group;
      const int64_t row = (int64_t)row0 + t;
      if (a.splits > 1) {
        const int64_t at = a.part_tokens > 0 ? (int64_t)s * a.part_tokens + t : row;
        float* part = a.partial + ((at * a.heads + head) * a.splits + split) * (HD + 4);
        *(float4_t*)(part + d) = o;
        if (d == 0) part[HD] = to, part[HD + 1] = total, part[HD + 2] = unit;
      } else {
        const float inv = total > 0.f || total != total ? 1.f / total : 0.f;
        uint16_t w[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const float x = B8 ? pa_times_power(o[k] * inv, unit) : o[k] * inv;
          w[k] = a.bf16 ? __builtin_bit_cast(uint16_t, (bf16_t)x) : __builtin_bit_cast(uint16_t, (half_t)x);
        }
        const int64_t at = a.out_mb > 0 ? packed_act_offset((int)row, head * HD + d, a.out_mb) : row * a.ldo + head * HD + d;
        *(pg_u2*)((uint16_t*)a.out + at) = pg_u2{(uint32_t)w[0] | (uint32_t)w[1] << 16, (uint32_t)w[2] | (uint32_t)w[3] << 16};
      }
    }
  }
}

// ---- portions of prompts: more than `few` rows (token, query head) of a key/value head in a sequence ----------------
// Workgroup = 128 rows, 4 waves of 32; tiles of 64 keys go through LDS, two of keys and two of values, one barrier a
// tile.  Everything transposed as above, with v_mfma 32x32x16: a lane has row n = lane % 32 and, with hl = lane / 32, 16 of 32
// keys.  Row m of a block of S^T stands for the key with bits 2 and 3 of m exchanged, so that the eight probabilities
// of a step of the product with V belong to eight consecutive keys: one 128-bit read of the transposed values.
// 16-bit pages go to LDS directly (global_load_lds_dwordx4: 16 bytes a lane to consecutive places, from anywhere), 8-bit
// ones through registers, where they become fp16: keys times 2^(e - the tile's largest e), values times 2^(e - E), E the largest so
// far, both exact while what is seen lies within 2^PT_NEAR of the largest; from the first tile on where it does not, codes stay
// as they are and exponents go into scores and probabilities, as above (PT_NEAR).  Chunks of 16 bytes of a row are exchanged
// by the row's number, so that reads of many rows meet all banks.
//
// Bound by the vector units beside the matrix cores: a wave's tile of 128 dimensions is 32 products of 32 cycles and, for
// 32 scores a lane, as many exponentials (16 cycles each) and some 150 other instructions, and the two waves that a SIMD
// holds overlap little of it; a short call by its longest workgroups too, all of which run at once.  Measured, heads of 128, a hundred
// calls in a row (short runs, at a higher clock), beside 1.50 PFLOP/s of a large fp16 product and 1.58 of bf16: 8192 tokens of 32 heads
// from the start, fp16, 550 GFLOP, 0.64 ms, 0.86 PFLOP/s; four portions of 304 to 513 tokens of 32 heads behind 1101 to 1536, 39.5
// GFLOP, 92 us, 0.43 (78, 0.51), 480 workgroups of 26 tiles on the average and 33 at most; bf16, portions of 4096 and 2324 tokens of 32
// heads on 8 with a window of 1024, 108 GFLOP, 198 us, 0.55 (181, 0.60; tiles at the window's ends are computed whole); the four portions in
// e4m3 115, in int8 118.  Tried without gain: the scheduler's group
// hints, wave priorities; without loads the kernel takes 0.9 of its time, without the product with V 0.87.
constexpr int PT_BM = 128, PT_BN = 64, PT_THREADS = 256;
// Exponents of keys of a tile, and of values so far, that rows of a workgroup see: up to so far apart one power of two for all
// serves.  (A code is a multiple of 2^-9 and at most 448, so that fp16 holds it times 2^-12 exactly; a probability below
// 2^-24 of the largest, which fp16 rounds to 2^-35, then is off by 2^-22 of what the largest adds.  us, four portions of 304 to
// 513 tokens of 32 heads of 128 behind 1101 to 1536: near e4m3 115, int8 118, far apart from the first tile on 148 and 136.)
constexpr int PT_NEAR = 12;

typedef __attribute__((address_space(3))) void pt_lds_void;

// where chunk c of row `row` of a tile with CH chunks to a row stands in that row
template <int CH>
__device__ __forceinline__ int pt_place(int c, int row) {
  if (CH % 16 == 0) return c ^ (row & 15);
  if (CH % 8 == 0) return c ^ ((row >> 1) & 7);
  const int p = c + (CH == 12 ? (row >> 2) & 3 : (row >> 3) & 1);  // 12, 10: 192, 160 bytes
  return p >= CH ? p - CH : p;
}
template <int CH>
__device__ __forceinline__ int pt_chunk_at(int p, int row) {  // the chunk that stands at place p
  if (CH % 8 == 0) return pt_place<CH>(p, row);
  const int c = p - (CH == 12 ? (row >> 2) & 3 : (row >> 3) & 1);
  return c < 0 ? c + CH : c;
}

// a pointer that is the same in all lanes, in scalar registers
__device__ __forceinline__ const char* pt_uniform(const char* p) {
  const uint64_t w = (uint64_t)p;
  const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)w), hi = __builtin_amdgcn_readfirstlane((uint32_t)(w >> 32));
  return (const char*)((uint64_t)hi << 32 | lo);
}

template <int F>
__device__ __forceinline__ float16_t pt_mfma(pg_u4 a, pg_u4 b, float16_t c) {
  if (F == PG_BF16)
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(half8_t, a), __builtin_bit_cast(half8_t, b), c, 0, 0, 0);
}

template <int F, int HD>
__global__ __launch_bounds__(PT_THREADS, HD <= 128 ? 2 : 1) void paged_tile_kernel(PagedAttention a) {
  typedef PaFormat<F> X;
  constexpr bool B8 = X::bits8;
  constexpr int ES = X::ES;
  constexpr int KSTEPS = HD / 16, DBLK = (HD + 31) / 32;
  constexpr int AHEAD = 2, VAHEAD = 2;  // fragments requested ahead: pairs of K, of V
  constexpr int CH = HD / 8;                    // 16-byte chunks of a key row in LDS, which holds 16-bit elements
  constexpr int ROWB = HD * 2, TILEB = PT_BN * ROWB;
  constexpr float SHIFT = X::SHIFT;
  extern __shared__ __attribute__((aligned(16))) char lds[];  // K, K, V, V

  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n32 = lane & 31, hl = lane >> 5;
  const int group = a.heads / a.kv_heads;
  // workgroup -> (sequence, key/value head), row block, split: see the launch
  int unit_id, rest;
  if (a.grouped) {
    const int j = blockIdx.x >> 3, per = a.row_blocks * a.splits;
    unit_id = (j / per) * 8 + (blockIdx.x & 7);
    rest = j % per;
  } else {
    const int units = a.nseq * a.kv_heads;
    rest = blockIdx.x / units;
    unit_id = blockIdx.x - rest * units;
  }
  const int split = rest % a.splits, rb = a.row_blocks - 1 - rest / a.splits;
  const int s = unit_id / a.kv_heads, h = unit_id - s * a.kv_heads;
  if (s >= a.nseq) return;
  const pg_uniform_i32* seq_start = (const pg_uniform_i32*)(uintptr_t)a.seq_start;
  const int row0 = seq_start[s], pos = ((const pg_uniform_i32*)(uintptr_t)a.seq_pos)[s];
  const int count = min(min(seq_start[s + 1], a.M) - row0, a.max_count);
  if (pos < 0 || row0 < 0 || count <= 0 || count * group <= a.few || rb * PT_BM >= count * group) return;
  const int page = 1 << a.page_log2, rows = count * group, rho0 = rb * PT_BM;
  const int limit = a.blocks * page - 1;
  auto position = [&](int rho) { return (int)min((int64_t)pos + min(rho, rows - 1) / group, (int64_t)limit); };
  const PaTiles<PT_BN> tiles(position(rho0), position(rho0 + PT_BM - 1), a.window, a.sinks);
  const int per = (tiles.n + a.splits - 1) / a.splits;
  const int it0 = split * per, it_end = min(tiles.n, it0 + per);
  // of this wave
  const int w0 = rho0 + wave * 32;
  const int p_lo = position(w0), p_hi = position(w0 + 31);

  // ---- queries: B operand, row n32, 8 dimensions at 16 ks + 8 hl ----
  const int rho = w0 + n32;
  const bool live = rho < rows;
  const int tok = live ? rho / group : 0, g = live ? rho - tok * group : 0;
  const int pn = live ? position(rho) : -1;
  pg_u4 qf[KSTEPS];
  const float qs = a.scale * PA_LOG2E;
  int eq = 0;  // 8 bits: the power of two that the row's queries stand for
  {
    const char* q = (const char*)a.q + (((int64_t)row0 + tok) * a.ldq + (int64_t)(h * group + g) * HD + hl * 8) * 2;
#pragma unroll
    for (int ks = 0; ks < KSTEPS; ++ks) qf[ks] = *(const pg_u4*)(q + ks * 32);
    if (B8 && a.bf16) {
      float big = 0.f;
#pragma unroll
      for (int ks = 0; ks < KSTEPS; ++ks) {
        const bf16x8_t v = __builtin_bit_cast(bf16x8_t, qf[ks]);
#pragma unroll
        for (int i = 0; i < 8; ++i) big = fmaxf(big, fabsf((float)v[i]));
      }
      big = fmaxf(big, __shfl_xor(big, 32, MSA_WAVE));
      const int k = min(max((int)(__builtin_bit_cast(uint32_t, big) >> 23) - 127 - 8, -118), 120);
#pragma unroll
      for (int ks = 0; ks < KSTEPS; ++ks) {
        const bf16x8_t v = __builtin_bit_cast(bf16x8_t, qf[ks]);
        half8_t w;
#pragma unroll
        for (int i = 0; i < 8; ++i) w[i] = (half_t)ldexpf((float)v[i], -k);
        qf[ks] = __builtin_bit_cast(pg_u4, w);
      }
      eq = k;
    }
  }

  // ---- tiles.  (The table is read through the scalar cache: a vector load would be waited for together with all the
  // loads to LDS in front of it) ----
  const pg_uniform_i32* table = (const pg_uniform_i32*)(uintptr_t)(a.table + (int64_t)s * a.table_stride);
  // entries of the pages of tile i's four groups of sixteen keys (one entry of pages of 64 and more), to be checked when they
  // are used: a check here would wait for them
  const bool large = a.page_log2 >= 6;
  auto entries = [&](int i) {
    const int key0 = tiles.tile(min(i, it_end - 1)) * PT_BN, last = a.blocks - 1;
    PtPages e;
    e.a = table[min(key0 >> a.page_log2, last)];
    e.b = e.c = e.d = e.a;
    if (!large) {
      e.b = table[min((key0 + 16) >> a.page_log2, last)];
      e.c = table[min((key0 + 32) >> a.page_log2, last)];
      e.d = table[min((key0 + 48) >> a.page_log2, last)];
    }
    return e;
  };
  auto checked = [&](PtPages e, int i) {
    const int key0 = tiles.tile(i) * PT_BN;
    auto one = [&](int pg, int key) { return (key >> a.page_log2) < a.blocks && (unsigned)pg < (unsigned)a.pages ? pg : -1; };
    return PtPages{one(e.a, key0), one(e.b, key0 + 16), one(e.c, key0 + 32), one(e.d, key0 + 48)};
  };
  const int64_t unit = (int64_t)page * HD * ES, page_bytes = unit * a.kv_heads;  // of a page and head, of a page
  const uint32_t lds0 = (uint32_t)(uintptr_t)(pt_lds_void*)lds;
  // 16 bits.  Keys: the sixteen of this wave, which are of one page, fill its sixteen rows of the tile.  Values: every
  // fourth group of eight rows (dimensions) is this wave's; a lane has the same chunk (eight keys) in all of them.
  constexpr int KI = (16 * CH + 63) / 64, VI = (HD / 8 + 3) / 4;
  uint32_t koff[B8 ? 1 : KI];
  const int vrow = wave * 8 + (lane >> 3), vc = pt_chunk_at<8>(lane & 7, vrow);
  if (!B8) {
#pragma unroll
    for (int u = 0; u < KI; ++u) {
      const int at = u * 64 + lane, row = min(at / CH, 15);
      koff[u] = row * ROWB + pt_chunk_at<CH>(at % CH, row) * 16;
    }
  }
  const char *k_head = (const char*)a.k_pages + h * unit, *v_lane = (const char*)a.v_pages + h * unit + vrow * page * 2;
  auto issue = [&](int i, int slot, PtPages pg) {
    const int key0 = tiles.tile(i) * PT_BN, in = page - 1;
    {
      const char* from = k_head + max(pg.of(wave), 0) * page_bytes + ((key0 + wave * 16) & in) * ROWB;
#pragma unroll
      for (int u = 0; u < KI; ++u) {
        const uint32_t la = lds0 + slot * TILEB + wave * 16 * ROWB + u * 1024;
        if ((u + 1) * 64 <= 16 * CH || lane < 16 * CH - u * 64)
          asm volatile("s_mov_b32 m0, %2\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(koff[u]), "s"(pt_uniform(from)), "s"(la) : "memory");
      }
    }
    const char* from = v_lane + max(pg.of(vc >> 1), 0) * page_bytes + ((key0 + vc * 8) & in) * 2;
#pragma unroll
    for (int u = 0; u < VI; ++u) {
      const uint32_t la = lds0 + (2 + slot) * TILEB + (u * 4 + wave) * 1024;
      if (HD % 32 == 0 || u * 4 + wave < HD / 8)
        asm volatile("s_mov_b32 m0, %1\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(from), "s"(la) : "memory");
      from += page * 64;
    }
  };
  // whether any row of the workgroup sees the key
  const int g_lo = position(rho0), g_hi = position(rho0 + PT_BM - 1);
  auto anyone = [&](int key) { return pa_seen<1>(key, g_lo, g_hi, a.window, a.sinks) != 0; };
  // 8 bits: chunks of 16 elements, registers in between.  Lane i of every wave has the exponents of key i; the factors that
  // follow from them reach the lanes that need them through LDS of the wave's own.
  constexpr int CB = HD / 16, KN = (PT_BN * CB + PT_THREADS - 1) / PT_THREADS, VN = (HD * 4 + PT_THREADS - 1) / PT_THREADS;
  __shared__ __attribute__((aligned(16))) int8_t s_exponent[B8 ? 2 : 1][B8 ? 64 : 1];
  __shared__ __attribute__((aligned(16))) half_t s_factor[B8 ? PT_THREADS / 64 : 1][2][64];
  // Addresses that follow from the thread's number are formed anew for each tile where registers end: kept across the loop they
  // would take others to scratch memory.  (us: 256 dimensions in int8 230 with all of them kept, 155 with those of the keys'
  // fragments, 141 with none; e4m3, which has the registers, 125 and 129; 128 dimensions 111 and 115)
  constexpr bool ANEW = F == PG_I8 && HD > 192;
  pg_u4 kr[B8 ? KN : 1], vr[B8 ? VN : 1];
  int ke = 0, ve = 0, least = 127;  // of the lane's key; least: of values so far
  const int vg = threadIdx.x & 3;       // the sixteen keys that the thread's chunks of V belong to
  auto fetch = [&](int i, PtPages pg) {
    const int key0 = tiles.tile(i) * PT_BN, in = page - 1;
    int tid = threadIdx.x;
    if (ANEW) asm volatile("" : "+v"(tid));
#pragma unroll
    for (int j = 0; j < KN; ++j) {
      const int at = min(tid + j * PT_THREADS, PT_BN * CB - 1), row = at / CB, c = at % CB;
      kr[j] = *(const pg_u4*)((const char*)a.k_pages + h * unit + max(pg.of(row >> 4), 0) * page_bytes + ((key0 + row) & in) * HD + c * 16);
    }
    const char* from = (const char*)a.v_pages + h * unit + max(pg.of(vg), 0) * page_bytes + ((key0 + vg * 16) & in);
#pragma unroll
    for (int j = 0; j < VN; ++j) vr[j] = *(const pg_u4*)(from + (min(tid + j * PT_THREADS, HD * 4 - 1) >> 2) * page);
    const int64_t ul = ((int64_t)max(pg.of(lane >> 4), 0) * a.kv_heads + h) * page + ((key0 + lane) & in);
    ke = a.k_exp[ul];
    ve = a.v_exp[ul];
  };
  auto wave_most = [](int v) { return __builtin_amdgcn_readfirstlane((int)wave_max((float)v)); };
  // ek, ev: the exponents that the tile's keys and values are relative to.  Returns whether some are further from them than
  // that allows (then the tile is no use).
  auto stage = [&](int i, int slot, PtPages pg, int& ek, int& ev) {
    const int key0 = tiles.tile(i) * PT_BN;
    int tid = threadIdx.x;
    if (ANEW) asm volatile("" : "+v"(tid));
    const bool mine = pg.of(lane >> 4) >= 0 && anyone(key0 + lane);
    ek = wave_most(mine ? ke : -127);
    ev = max(ev, wave_most(mine ? ve : -127));
    least = min(least, mine ? ve : 127);
    const uint64_t beyond = __ballot((mine && ke < ek - PT_NEAR) || least < ev - PT_NEAR);
    // 2^(e - largest); 0 below what fp16 can be (keys that nobody sees)
    auto factor = [](int e) { return e < -24 ? (half_t)0.f : (half_t)__builtin_bit_cast(float, (uint32_t)(127 + min(e, 0)) << 23); };
    s_factor[wave][0][lane] = factor(ke - ek);
    s_factor[wave][1][lane] = factor(ve - ev);
    char* kt = lds + slot * TILEB;
    char* vt = lds + (2 + slot) * TILEB;
#pragma unroll
    for (int j = 0; j < KN; ++j) {
      const int at = tid + j * PT_THREADS, row = at / CB, c = at % CB;
      if ((PT_BN * CB) % PT_THREADS == 0 || at < PT_BN * CB) {
        const half_t f = s_factor[wave][0][row & 63];
#pragma unroll
        for (int e = 0; e < 2; ++e)
          *(half8_t*)(kt + row * ROWB + pt_place<CH>(2 * c + e, row) * 16) = __builtin_bit_cast(half8_t, pa_operand<F>(kr[j], e)) * f;
      }
    }
    const half8_t f[2] = {*(const half8_t*)&s_factor[wave][1][vg * 16], *(const half8_t*)&s_factor[wave][1][vg * 16 + 8]};
    const uint32_t seen = pg.of(vg) >= 0 ? pa_seen<16>(key0 + vg * 16, g_lo, g_hi, a.window, a.sinks) : 0;
#pragma unroll
    for (int j = 0; j < VN; ++j) {
      const int at = tid + j * PT_THREADS, row = at >> 2;
      if ((HD * 4) % PT_THREADS == 0 || at < HD * 4) {
        pg_u4 w = vr[j];
        if (seen != 0xffff) {
#pragma unroll
          for (int k = 0; k < 4; ++k) w[k] = pa_keep<F>(w[k], seen >> (4 * k));
        }
#pragma unroll
        for (int e = 0; e < 2; ++e)
          *(half8_t*)(vt + row * 128 + pt_place<8>(2 * vg + e, row) * 16) = __builtin_bit_cast(half8_t, pa_operand<F>(w, e)) * f[e];
      }
    }
    return beyond != 0;
  };

  // ---- fragments: K block ib, step ks: row with bits 2 and 3 of n32 exchanged, chunk 2 ks + hl.  V^T block db, step c (16
  // keys): row 32 db + n32, chunk 2 c + hl ----
  const int krow = (n32 & ~12) | ((n32 & 4) << 1) | ((n32 & 8) >> 1);
  auto v_at = [&](const char* vt, int db, int st) {
    const int row = HD % 32 == 0 ? db * 32 + n32 : min(db * 32 + n32, HD - 1);
    return *(const pg_u4*)(vt + row * 128 + pt_place<8>(2 * st + hl, row) * 16);
  };
  constexpr int G = F == PG_BF16 ? PG_BF16 : PG_F16;  // LDS holds 16 bits in every format
  const float16_t zero16 = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  float16_t o[DBLK];
#pragma unroll
  for (int d = 0; d < DBLK; ++d) o[d] = zero16;
  float m = -INFINITY, l = 0.f;
  int E = -127, ek = 0, ev = -127;  // what the accumulators are relative to, and this tile's keys and values
  bool far = false;
  PtPages pg = {-1, -1, -1, -1}, next = pg;  // this tile's, and entries of the next one's
  if (it0 < it_end) {
    pg = checked(entries(it0), it0);
    next = entries(it0 + 1);
    if (B8) {
      fetch(it0, pg);
      far = stage(it0, 0, pg, ek, ev);
    } else {
      issue(it0, 0, pg);
    }
  }
  // (the queries have arrived from here on: the compiler, which does not count the loads to LDS, would wait for them in the
  // loop, and with them for the tile just requested)
#pragma unroll
  for (int ks = 0; ks < KSTEPS; ++ks) asm volatile("" : "+v"(qf[ks]));
  int i = it0;
  for (; i < it_end && !far; ++i) {
    const int slot = (i - it0) & 1;
    const int here = (pg.a >= 0 ? 1 : 0) | (pg.b >= 0 ? 2 : 0) | (pg.c >= 0 ? 4 : 0) | (pg.d >= 0 ? 8 : 0);
    if (!B8) asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();  // the tile is complete, and the other slots are free
    if (i + 1 < it_end) {
      pg = checked(next, i + 1);
      if (B8) fetch(i + 1, pg);
      else issue(i + 1, slot ^ 1, pg);
    }
    const char* kt = lds + slot * TILEB;
    char* vt = lds + (2 + slot) * TILEB;
    const int key0 = tiles.tile(i) * PT_BN;
    const bool whole = key0 + PT_BN - 1 <= p_lo && (a.window <= 0 || key0 > p_hi - a.window || key0 + PT_BN <= a.sinks) && here == 15;
    // Tiles of which not every row sees every key (of the workgroup): values of keys that no row sees may be anything and
    // become zeros.  Whether there is one then that is not finite: it must reach the rows that see it only (0 times
    // infinity is NaN), so it is added to those and left out of the product.
    bool odd = false;
    if (F != PG_I8 && !(key0 + PT_BN - 1 <= g_lo && (a.window <= 0 || key0 > g_hi - a.window || key0 + PT_BN <= a.sinks) && here == 15)) {
      typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
      u16x2 most = {0, 0};
#pragma unroll 1
      for (int at = threadIdx.x; at < HD * 8; at += PT_THREADS) {
        const int key = key0 + pt_chunk_at<8>(at & 7, at >> 3) * 8;
        const uint32_t seen = (here >> ((key - key0) >> 4)) & 1 ? pa_seen<8>(key, g_lo, g_hi, a.window, a.sinks) : 0;
        pg_u4 v = *(pg_u4*)(vt + at * 16);
        if (seen != 255) {
#pragma unroll
          for (int k = 0; k < 4; ++k) v[k] = pa_keep<G>(v[k], seen >> (2 * k));
          *(pg_u4*)(vt + at * 16) = v;
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) most = __builtin_elementwise_max(most, __builtin_bit_cast(u16x2, v[k] & 0x7fff7fffu));
      }
      odd = max(most[0], most[1]) >= (G == PG_BF16 ? 0x7f80 : 0x7c00);
      odd = __syncthreads_or(odd);
    }
    // (a wave whose rows see nothing of the tile has nothing to do)
    const bool none = key0 > p_hi || w0 >= rows || (a.window > 0 && key0 + PT_BN - 1 <= p_lo - a.window && key0 >= a.sinks);
    // (zeros have the least exponent there is, queries of zeros too: below what fp32 can be any score is zero, but those of keys
    // that are not seen are -infinity, which a factor of zero would make NaN; above it a product of zero stays one)
    const float to_score = B8 ? fminf(fmaxf(ldexpf(qs, ek + eq), FLT_MIN), FLT_MAX) : qs;
    // Two copies: tiles that every row of the wave sees whole, and others.
    auto attend = [&](auto edge) {
      constexpr bool EDGE = decltype(edge)::value;
      // (the order below is kept: left alone, the compiler requests a fragment right before its product and waits for it)
      float16_t sc[2];
      pg_u4 kf[AHEAD][2], vf[VAHEAD];
      int krow_here = krow, half = hl;
      if (ANEW) asm volatile("" : "+v"(krow_here), "+v"(half));
      auto k_at = [&](int ks, int ib) {
        const int row = ib * 32 + krow_here;
        return *(const pg_u4*)(kt + row * ROWB + pt_place<CH>(2 * ks + half, row) * 16);
      };
#pragma unroll
      for (int ks = 0; ks < AHEAD; ++ks) kf[ks][0] = k_at(ks, 0), kf[ks][1] = k_at(ks, 1);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int ks = 0; ks < KSTEPS; ++ks) {
#pragma unroll
        for (int ib = 0; ib < 2; ++ib) {
          sc[ib] = pt_mfma<F>(kf[ks % AHEAD][ib], qf[ks], ks == 0 ? zero16 : sc[ib]);
          if (ks + AHEAD < KSTEPS) kf[ks % AHEAD][ib] = k_at(ks + AHEAD, ib);
        }
        __builtin_amdgcn_sched_barrier(0);
      }
#pragma unroll
      for (int n = 0; n < VAHEAD; ++n) vf[n] = v_at(vt, n % DBLK, n / DBLK);
      __builtin_amdgcn_sched_barrier(0);
      float z[32];  // keys key0 + 16 (j / 8) + 8 hl + j % 8
#pragma unroll
      for (int j = 0; j < 32; ++j) z[j] = sc[j >> 4][j & 15];
      uint32_t sees = ~0u;  // of those keys, the row's
      if (EDGE) {
        sees = 0;
#pragma unroll
        for (int g8 = 0; g8 < 4; ++g8)
          sees |= pa_seen<8>(key0 + g8 * 16 + hl * 8, pn, pn, a.window, a.sinks) * ((here >> g8) & 1) << (g8 * 8);
#pragma unroll
        for (int j = 0; j < 32; ++j) z[j] = (sees >> j) & 1 ? z[j] : -INFINITY;
      }
      float top = z[0];
#pragma unroll
      for (int j = 1; j < 32; ++j) top = fmaxf(top, z[j]);
      top *= to_score;
      if (B8 && ev > E) {
#pragma unroll
        for (int d = 0; d < DBLK; ++d)
#pragma unroll
          for (int v = 0; v < 16; ++v) o[d][v] = ldexpf(o[d][v], E - ev);
        E = ev;
      }
      if (__ballot(top > m + PA_LAZY)) {
        const float to = fmaxf(m, fmaxf(top, __shfl_xor(top, 32, MSA_WAVE)));
        const float w = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - to);
        m = to;
        l *= w;
#pragma unroll
        for (int d = 0; d < DBLK; ++d)
#pragma unroll
          for (int v = 0; v < 16; ++v) o[d][v] *= w;
      }
      float c = to_score, off;
      pa_relative(z, c, off, m, SHIFT);
      pg_u4 p[4];  // steps of sixteen keys of the product with V
      float sum[2] = {0.f, 0.f};  // of the probabilities as they are rounded: weights that add up to one
      auto pair = [&](int st, int j) {
        const float e0 = __builtin_amdgcn_exp2f(__builtin_fmaf(z[st * 8 + 2 * j], c, -off));
        const float e1 = __builtin_amdgcn_exp2f(__builtin_fmaf(z[st * 8 + 2 * j + 1], c, -off));
        if (F == PG_BF16) {
          const bf16x2_t w = {(bf16_t)e0, (bf16_t)e1}, one = {(bf16_t)1.f, (bf16_t)1.f};
          sum[j & 1] = __builtin_amdgcn_fdot2_f32_bf16(w, one, sum[j & 1], false);
          p[st][j] = __builtin_bit_cast(uint32_t, w);
        } else {
          const half2_t w = {(half_t)e0, (half_t)e1}, one = {(half_t)1.f, (half_t)1.f};
          sum[j & 1] = __builtin_amdgcn_fdot2(w, one, sum[j & 1], false);
          p[st][j] = __builtin_bit_cast(uint32_t, w);
        }
      };
      if (EDGE && F != PG_I8) {
        if (odd) {  // (an infinity or a NaN times a probability is itself)
#pragma unroll 1
          for (int j = 0; j < PT_BN; ++j) {
            int hl4 = hl * 4;  // (formed anew: 64 addresses would be kept through both loops)
            asm volatile("" : "+v"(hl4));
            const bool mine = (pa_seen<1>(key0 + j, pn, pn, a.window, a.sinks) & (here >> (j >> 4))) != 0;
#pragma unroll
            for (int db = 0; db < DBLK; ++db)
#pragma unroll
              for (int v = 0; v < 16; ++v) {
                const int row = min(db * 32 + (v >> 2) * 8 + hl4 + (v & 3), HD - 1);
                const uint32_t x = *(const uint16_t*)(vt + row * 128 + pt_place<8>(j >> 3, row) * 16 + (j & 7) * 2);
                const float f = G == PG_BF16 ? __builtin_bit_cast(float, x << 16) : (float)__builtin_bit_cast(half_t, (uint16_t)x);
                o[db][v] += (mine & !(fabsf(f) < INFINITY)) ? f : 0.f;
              }
          }
        }
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) pair(0, j);
#pragma unroll
      for (int st = 0; st < 4; ++st) {
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int db = 0; db < DBLK; ++db) {
          const int n = st * DBLK + db;
          pg_u4 v = vf[n % VAHEAD];
          if (EDGE && F != PG_I8) {
            if (odd) {
#pragma unroll
              for (int k = 0; k < 4; ++k) v[k] = pa_finite<G>(v[k]);
            }
          }
          o[db] = pt_mfma<F>(v, p[st], o[db]);
          if (n + VAHEAD < 4 * DBLK) vf[n % VAHEAD] = v_at(vt, (n + VAHEAD) % DBLK, (n + VAHEAD) / DBLK);
          if (st < 3) {
#pragma unroll
            for (int j = 0; j < 4; ++j)
              if (db == (DBLK > 4 ? j : j * DBLK / 4)) pair(st + 1, j);
          }
          __builtin_amdgcn_sched_barrier(0);
        }
      }
      l += sum[0] + sum[1];
    };
    if (whole) attend(std::false_type{});
    else if (!none) attend(std::true_type{});
    if (B8 && i + 1 < it_end) far = stage(i + 1, slot ^ 1, pg, ek, ev);
    next = entries(i + 2);
  }

  // ---- 8 bits, exponents far apart: codes in LDS, every key's exponent in its score, every value's in its probability, relative
  // to the row's own running maximum R as in the kernel above; one tile at a time ----
  float power = B8 ? (float)E : 0.f;  // the accumulators are in units of 2^power
  if constexpr (B8) {
    float R = m == -INFINITY ? -INFINITY : (float)E;
    // (what follows from the thread's number is formed here, not in front of the loop above, which needs the registers)
    int tid = threadIdx.x;
    asm volatile("" : "+v"(tid));
    const int n32 = tid & 31, hl = (tid >> 5) & 1, krow = (n32 & ~12) | ((n32 & 4) << 1) | ((n32 & 8) >> 1);
    for (; i < it_end; ++i) {
      const int key0 = tiles.tile(i) * PT_BN;
      const int here = (pg.a >= 0 ? 1 : 0) | (pg.b >= 0 ? 2 : 0) | (pg.c >= 0 ? 4 : 0) | (pg.d >= 0 ? 8 : 0);
      fetch(i, pg);
      __syncthreads();  // the tile before has been read
      bool odd = false;
#pragma unroll
      for (int j = 0; j < KN; ++j) {
        const int at = tid + j * PT_THREADS, row = at / CB, c = at % CB;
        if ((PT_BN * CB) % PT_THREADS == 0 || at < PT_BN * CB) {
#pragma unroll
          for (int e = 0; e < 2; ++e) *(pg_u4*)(lds + row * ROWB + pt_place<CH>(2 * c + e, row) * 16) = pa_operand<F>(kr[j], e);
        }
      }
      char* vt = lds + 2 * TILEB;
      const uint32_t seen = pg.of(vg) >= 0 ? pa_seen<16>(key0 + vg * 16, g_lo, g_hi, a.window, a.sinks) : 0;
#pragma unroll
      for (int j = 0; j < VN; ++j) {
        const int at = tid + j * PT_THREADS, row = at >> 2;
        if ((HD * 4) % PT_THREADS == 0 || at < HD * 4) {
          pg_u4 w = vr[j];
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            w[k] = pa_keep<F>(w[k], seen >> (4 * k));
            odd |= pa_not_finite<F>(w[k], 0) != 0;
          }
#pragma unroll
          for (int e = 0; e < 2; ++e) *(pg_u4*)(vt + row * 128 + pt_place<8>(2 * vg + e, row) * 16) = pa_operand<F>(w, e);
        }
      }
      if (wave == 0) s_exponent[0][tid] = (int8_t)ke, s_exponent[1][tid] = (int8_t)ve;
      odd = __syncthreads_or(odd);  // the tile is complete
      if (i + 1 < it_end) pg = checked(next, i + 1);
      next = entries(i + 2);
      if (key0 > p_hi || w0 >= rows) continue;
      float z[32], c = qs, off;
      {
        float16_t sc[2];
#pragma unroll
        for (int ks = 0; ks < KSTEPS; ++ks)
#pragma unroll
          for (int ib = 0; ib < 2; ++ib) {
            const int row = ib * 32 + krow;
            sc[ib] = pt_mfma<F>(*(const pg_u4*)(lds + row * ROWB + pt_place<CH>(2 * ks + hl, row) * 16), qf[ks], ks == 0 ? zero16 : sc[ib]);
          }
#pragma unroll
        for (int j = 0; j < 32; ++j) z[j] = sc[j >> 4][j & 15];
      }
      auto exponent = [](pg_u2 w, int j) { return (int)(int8_t)(w[j >> 2] >> ((j & 3) * 8)); };
      float top = -INFINITY;
#pragma unroll
      for (int g8 = 0; g8 < 4; ++g8) {
        const pg_u2 x = *(const pg_u2*)&s_exponent[0][g8 * 16 + hl * 8];
        const uint32_t sees = pa_seen<8>(key0 + g8 * 16 + hl * 8, pn, pn, a.window, a.sinks) * ((here >> g8) & 1);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          float& s = z[g8 * 8 + j];
          s = (sees >> j) & 1 ? ldexpf(s, exponent(x, j) + eq) : -INFINITY;
          top = fmaxf(top, s);
        }
      }
      top *= qs;
      if (__ballot(top > m + PA_LAZY)) {
        const float to = fmaxf(m, fmaxf(top, __shfl_xor(top, 32, MSA_WAVE)));
        l *= m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - to);
        R -= m == -INFINITY ? 0.f : to - m;
        m = to;
      }
      pa_relative(z, c, off, m, 0.f);
      float sum = 0.f, most = -INFINITY;
#pragma unroll
      for (int g8 = 0; g8 < 4; ++g8) {
        const pg_u2 x = *(const pg_u2*)&s_exponent[1][g8 * 16 + hl * 8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          float& s = z[g8 * 8 + j];
          s = __builtin_fmaf(s, c, -off);
          sum += __builtin_amdgcn_exp2f(s + SHIFT);
          s += (float)exponent(x, j);
          most = fmaxf(most, s);
        }
      }
      l += sum;
      if (__ballot(most > R + PA_LAZY)) {
        const float to = fmaxf(R, fmaxf(most, __shfl_xor(most, 32, MSA_WAVE)));
        const float w = R == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(R - to);
        R = to;
#pragma unroll
        for (int d = 0; d < DBLK; ++d)
#pragma unroll
          for (int v = 0; v < 16; ++v) o[d][v] *= w;
      }
      if (F == PG_E4M3 && odd) {
#pragma unroll 1
        for (int j = 0; j < PT_BN; ++j) {
          const bool mine = (pa_seen<1>(key0 + j, pn, pn, a.window, a.sinks) & (here >> (j >> 4))) != 0;
          int hl4 = hl * 4;
          asm volatile("" : "+v"(hl4));
#pragma unroll
          for (int db = 0; db < DBLK; ++db)
#pragma unroll
            for (int v = 0; v < 16; ++v) {
              const int row = min(db * 32 + (v >> 2) * 8 + hl4 + (v & 3), HD - 1);
              const uint16_t x = *(const uint16_t*)(vt + row * 128 + pt_place<8>(j >> 3, row) * 16 + (j & 7) * 2);
              o[db][v] += mine && (x & 0x7fff) > 0x7c00 ? NAN : 0.f;
            }
        }
      }
      const float from = (R == -INFINITY ? 0.f : R) - SHIFT;
#pragma unroll
      for (int st = 0; st < 4; ++st) {
        pg_u4 p;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const half2_t w = {(half_t)__builtin_amdgcn_exp2f(z[st * 8 + 2 * j] - from), (half_t)__builtin_amdgcn_exp2f(z[st * 8 + 2 * j + 1] - from)};
          p[j] = __builtin_bit_cast(uint32_t, w);
        }
#pragma unroll
        for (int db = 0; db < DBLK; ++db) {
          const int row = min(db * 32 + n32, HD - 1);
          pg_u4 v = *(const pg_u4*)(vt + row * 128 + pt_place<8>(2 * st + hl, row) * 16);
          if (F == PG_E4M3 && odd) {
#pragma unroll
            for (int k = 0; k < 4; ++k) v[k] = pa_finite<G>(v[k]);
          }
          o[db] = pt_mfma<F>(v, p, o[db]);
        }
      }
    }
    if (far) power = R == -INFINITY ? 0.f : R;
  }

  // ---- O^T: row n32, dimensions 32 db + 8 blk + 4 hl + r ----
  l += __shfl_xor(l, 32, MSA_WAVE);
  if (!live) return;
  const int head = h * group + g;
  const int64_t row = (int64_t)row0 + tok;
  if (a.splits > 1) {
    float* to = a.partial + ((row * a.heads + head) * a.splits + split) * (HD + 4);
#pragma unroll
    for (int db = 0; db < DBLK; ++db)
#pragma unroll
      for (int blk = 0; blk < 4; ++blk) {
        const int d = db * 32 + blk * 8 + hl * 4;
        float4_t v;
#pragma unroll
        for (int r = 0; r < 4; ++r) v[r] = o[db][blk * 4 + r];
        if (HD % 32 == 0 || d < HD) *(float4_t*)(to + d) = v;
      }
    if (hl == 0) to[HD] = m, to[HD + 1] = l, to[HD + 2] = power;
    return;
  }
  const float inv = l > 0.f || l != l ? 1.f / l : 0.f;
#pragma unroll
  for (int db = 0; db < DBLK; ++db)
#pragma unroll
    for (int blk = 0; blk < 4; ++blk) {
      const int d = db * 32 + blk * 8 + hl * 4;
      uint16_t w[4];
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const float z = B8 ? pa_times_power(o[db][blk * 4 + r] * inv, power) : o[db][blk * 4 + r] * inv;
        w[r] = a.bf16 ? __builtin_bit_cast(uint16_t, (bf16_t)z) : __builtin_bit_cast(uint16_t, (half_t)z);
      }
      const int64_t at = a.out_mb > 0 ? packed_act_offset((int)row, head * HD + d, a.out_mb) : row * a.ldo + head * HD + d;
      if (HD % 32 == 0 || d < HD) *(pg_u2*)((uint16_t*)a.out + at) = pg_u2{(uint32_t)w[0] | (uint32_t)w[1] << 16, (uint32_t)w[2] | (uint32_t)w[3] << 16};
    }
}

template <int F, int HD>
bool pa_launch_tiles(const PagedAttention& a, hipStream_t stream) {
  constexpr int bytes = 4 * PT_BN * HD * 2;
  static std::atomic<uint64_t> done{0};
  if (!raise_lds((const void*)paged_tile_kernel<F, HD>, bytes, done)) return false;
  const int64_t units = (int64_t)a.nseq * a.kv_heads, per = (int64_t)a.row_blocks * a.splits;
  const int64_t n = a.grouped ? (units + 7) / 8 * 8 * per : units * per;
  hipLaunchKernelGGL((paged_tile_kernel<F, HD>), dim3((unsigned)n), dim3(PT_THREADS), bytes, stream, a);
  return true;
}

template <int F, int HD>
void pa_launch_rows(const PagedAttention& a, int rt, hipStream_t stream) {
  const dim3 grid((unsigned)((int64_t)a.nseq * a.row_blocks * a.kv_heads), (unsigned)a.splits);
  if (rt == 1) hipLaunchKernelGGL((paged_rows_kernel<F, HD, 1>), grid, dim3(PA_NW * 64), 0, stream, a);
  else hipLaunchKernelGGL((paged_rows_kernel<F, HD, 2>), grid, dim3(PA_NW * 64), 0, stream, a);
}

template <int F>
void pa_launch_rows_of(const PagedAttention& a, int hd, int rt, hipStream_t stream) {
  switch (hd) {
    case 64: return pa_launch_rows<F, 64>(a, rt, stream);
    case 80: return pa_launch_rows<F, 80>(a, rt, stream);
    case 96: return pa_launch_rows<F, 96>(a, rt, stream);
    case 128: return pa_launch_rows<F, 128>(a, rt, stream);
    case 192: return pa_launch_rows<F, 192>(a, rt, stream);
    default: return pa_launch_rows<F, 256>(a, rt, stream);
  }
}

template <int F>
bool pa_launch_tiles_of(const PagedAttention& a, int hd, hipStream_t stream) {
  switch (hd) {
    case 64: return pa_launch_tiles<F, 64>(a, stream);
    case 80: return pa_launch_tiles<F, 80>(a, stream);
    case 96: return pa_launch_tiles<F, 96>(a, stream);
    case 128: return pa_launch_tiles<F, 128>(a, stream);
    case 192: return pa_launch_tiles<F, 192>(a, stream);
    default: return pa_launch_tiles<F, 256>(a, stream);
  }
}

}  // namespace
