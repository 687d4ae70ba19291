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
// 8 bits: a code is exact in fp16.  The key's exponent scales the score; the value's goes into the probability, relative to the
// largest exponent E met so far (the accumulators are in units of 2^E), in fp32, before it is rounded.
#pragma once

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

__device__ __forceinline__ float pa_quads_max(float v) {
  v = fmaxf(v, __shfl_xor(v, 16, MSA_WAVE));
  return fmaxf(v, __shfl_xor(v, 32, MSA_WAVE));
}
__device__ __forceinline__ float pa_quads_sum(float v) {
  v += __shfl_xor(v, 16, MSA_WAVE);
  return v + __shfl_xor(v, 32, MSA_WAVE);
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
  __shared__ float s_m[PA_NW][16], s_l[PA_NW][16];

  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n16 = lane & 15, quad = lane >> 4;
  const int s = blockIdx.x / a.row_blocks, rb = blockIdx.x - s * a.row_blocks;
  const int h = blockIdx.y, split = blockIdx.z;
  const int group = a.heads / a.kv_heads;
  const int row0 = a.seq_start[s], pos = a.seq_pos[s];
  int count = min(a.seq_start[s + 1], a.M) - row0;
  count = min(count, a.max_count);
  if (pos < 0 || row0 < 0 || count <= 0 || rb * 16 * RT >= count * group) return;
  const int page = 1 << a.page_log2, rows = count * group, rho0 = rb * 16 * RT;
  const int limit = a.blocks * page - 1;  // last position that can be anywhere
  const int p_lo = (int)min((int64_t)pos + rho0 / group, (int64_t)limit);
  const int p_hi = (int)min((int64_t)pos + (min(rho0 + 16 * RT, rows) - 1) / group, (int64_t)limit);
  const PaTiles<KT> tiles(p_lo, p_hi, a.window, a.sinks);
  // this split's tiles, every PA_NW-th of them this wave's
  const int per = (tiles.n + a.splits - 1) / a.splits;
  const int it_end = min(tiles.n, (split + 1) * per);

  // ---- queries: B operand, row n16 of row tile rt, the dimensions that the lane's loads of K have ----
  pg_u4 qf[RT][KL][HALVES];
  float qs[RT];  // what turns a product into a score in log2 units
  int pn[RT];    // the row's position; rows past the last one see nothing
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    const int rho = rho0 + rt * 16 + n16;
    const bool live = rho < rows;
    const int t = live ? rho / group : 0, g = live ? rho - t * group : 0;
    pn[rt] = live ? (int)min((int64_t)pos + t, (int64_t)limit) : -1;
    const char* q = (const char*)a.q + (((int64_t)row0 + t) * a.ldq + (int64_t)(h * group + g) * HD) * 2;
    qs[rt] = a.scale * PA_LOG2E;
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
      qs[rt] = ldexpf(qs[rt], k);
    }
  }

  float4_t acc[RT][DT];
  float m[RT], l[RT];
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    m[rt] = -INFINITY;
    l[rt] = 0.f;
#pragma unroll
    for (int d = 0; d < DT; ++d) acc[rt][d] = float4_t{0.f, 0.f, 0.f, 0.f};
  }
  int E = -127;  // largest exponent of values met (8 bits)

  // ---- where tile i's keys are.  As a source of K a lane has keys of quad n16 / 4, as one of V of its own quad ----
  const int32_t* table = a.table + (int64_t)s * a.table_stride;
  auto look = [&](int i, int q) {  // page of quad q's keys of tile i (clamped past the end: those are masked)
    const int block = (tiles.tile(i) * KT + q * KQ) >> a.page_log2;
    return block < a.blocks ? table[block] : -1;
  };
  const int64_t unit = (int64_t)page * HD * ES;  // bytes of a page and head
  pg_u4 kf[NT][KL], vf[DT];
  auto load_k = [&](int i, int pg) {
    const int key = tiles.tile(i) * KT + (n16 >> 2) * KQ + (n16 & 3);
    const int64_t at = ((int64_t)(pg >= 0 && pg < a.pages ? pg : 0) * a.kv_heads + h) * unit + (int64_t)(key & (page - 1)) * (HD * ES) + quad * 16;
    const char* base = (const char*)a.k_pages + at;
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int c = 0; c < KL; ++c)
        kf[t][c] = (c + 1) * CD <= HD || quad * (CD / 4) + c * CD < HD
                       ? __builtin_nontemporal_load((const pg_u4*)(base + t * 4 * HD * ES + c * 64))
                       : pg_u4{0, 0, 0, 0};
  };
  auto load_v = [&](int i, int pg) {
    const int key = tiles.tile(i) * KT + quad * KQ;
    const int64_t at = ((int64_t)(pg >= 0 && pg < a.pages ? pg : 0) * a.kv_heads + h) * unit + ((int64_t)n16 * page + (key & (page - 1))) * ES;
    const char* base = (const char*)a.v_pages + at;
#pragma unroll
    for (int d = 0; d < DT; ++d) vf[d] = __builtin_nontemporal_load((const pg_u4*)(base + (int64_t)d * 16 * page * ES));
  };
  // exponents of the quad's keys
  pg_u4 kx, vx;
  auto load_x = [&](int i, int pg) {
    const int key = tiles.tile(i) * KT + quad * KQ;
    const int64_t at = ((int64_t)(pg >= 0 && pg < a.pages ? pg : 0) * a.kv_heads + h) * page + (key & (page - 1));
    kx = *(const pg_u4*)(a.k_exp + at);
    vx = *(const pg_u4*)(a.v_exp + at);
  };
  auto byte_of = [](pg_u4 w, int i) { return (int)(int8_t)(w[i >> 2] >> ((i & 3) * 8)); };

  for (int i = split * per + wave; i < it_end; i += PA_NW) {
    const int pk = look(i, n16 >> 2), pv = look(i, quad);
    load_k(i, pk);
    load_v(i, pv);
    if (B8) load_x(i, pv);
    const int key0 = tiles.tile(i) * KT;  // of the tile
    const int kq = key0 + quad * KQ;      // of the quad
    const bool here = pv >= 0 && pv < a.pages;
    // every row sees every key of the tile
    const bool whole = key0 + KT - 1 <= p_lo && (a.window <= 0 || key0 > p_hi - a.window || key0 + KT <= a.sinks) &&
                       __ballot(!here) == 0;
    // whether any row sees the key
    auto any_sees = [&](int key) {
      return here && key <= p_hi && (a.window <= 0 || key > p_lo - a.window || key < a.sinks);
    };
    if (B8) {
      int most = -127;
#pragma unroll
      for (int j = 0; j < KQ; ++j)
        if (whole || any_sees(kq + j)) most = max(most, byte_of(vx, j));
      if (__ballot(most > E)) {
        most = max(most, __shfl_xor(most, 16, MSA_WAVE));
        most = max(most, __shfl_xor(most, 32, MSA_WAVE));
        const int to = max(E, __builtin_amdgcn_readfirstlane(most));
#pragma unroll
        for (int rt = 0; rt < RT; ++rt)
#pragma unroll
          for (int d = 0; d < DT; ++d)
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[rt][d][e] = ldexpf(acc[rt][d][e], E - to);
        E = to;
      }
    }
    pg_u4 pf[RT][HALVES];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      float4_t sc[NT];
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        sc[t] = float4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int c = 0; c < KL; ++c)
#pragma unroll
          for (int e = 0; e < HALVES; ++e) sc[t] = pa_mfma<F>(pa_operand<F>(kf[t][c], e), qf[rt][c][e], sc[t]);
      }
      float top = -INFINITY;
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int j = t * 4 + e, key = kq + j;
          float z = sc[t][e] * qs[rt];
          if (B8) z = ldexpf(z, byte_of(kx, j));
          if (!whole && !(here && key <= pn[rt] && (a.window <= 0 || key > pn[rt] - a.window || key < a.sinks))) z = -INFINITY;
          sc[t][e] = z;
          top = fmaxf(top, z);
        }
      if (__ballot(top > m[rt] + PA_LAZY)) {  // (m = -inf: any score)
        const float to = fmaxf(m[rt], pa_quads_max(top));
        const float w = m[rt] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m[rt] - to);
        m[rt] = to;
        l[rt] *= w;
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[rt][d][e] *= w;
      }
      const float off = m[rt] == -INFINITY ? 0.f : m[rt];
      float p[KQ], sum = 0.f;
#pragma unroll
      for (int j = 0; j < KQ; ++j) {
        p[j] = __builtin_amdgcn_exp2f(sc[j >> 2][j & 3] - off);
        sum += p[j];
        if (B8) p[j] = ldexpf(p[j], (whole || any_sees(kq + j) ? byte_of(vx, j) : -127) - E + (int)X::SHIFT);
        else if (X::SHIFT != 0.f) p[j] *= exp2f(X::SHIFT);
      }
      l[rt] += sum;
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
    if (!whole) {
      // Keys that no row sees may hold anything: their values are taken as zeros.  A value that is not finite at a key
      // that some rows see and others do not must reach those rows only (0 times infinity is NaN): it is left out of
      // the product, and products with ones in the places of infinities and NaN say which rows it reaches.
      uint32_t seen = 0;
#pragma unroll
      for (int j = 0; j < KQ; ++j) seen |= any_sees(kq + j) ? 1u << j : 0;
      bool odd = false;
#pragma unroll
      for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          vf[d][i] = pa_keep<F>(vf[d][i], seen >> (i * (KQ / 4)));
          odd |= pa_not_finite<F>(vf[d][i], 0) != 0;
        }
      if (__ballot(odd)) {
#pragma unroll
        for (int d = 0; d < DT; ++d) {
#pragma unroll 1
          for (int kind = 1; kind <= 3; ++kind) {
            pg_u4 ones;
#pragma unroll
            for (int i = 0; i < 4; ++i) ones[i] = pa_not_finite<F>(vf[d][i], kind);
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) {
              float4_t hit = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
              for (int e = 0; e < HALVES; ++e) hit = pa_mfma<F>(pa_operand<F>(ones, e), pf[rt][e], hit);
#pragma unroll
              for (int i = 0; i < 4; ++i)
                if (hit[i] != 0.f) acc[rt][d][i] += kind == 1 ? INFINITY : kind == 2 ? -INFINITY : NAN;
            }
          }
#pragma unroll
          for (int i = 0; i < 4; ++i) vf[d][i] = pa_finite<F>(vf[d][i]);
        }
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
  }

  // ---- the waves' sums: one row tile at a time through LDS, added in the waves' order ----
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    const int left = min(16, rows - rho0 - rt * 16);
    if (left <= 0) break;
    l[rt] = pa_quads_sum(l[rt]);
    if (rt > 0) __syncthreads();
    if (quad == 0) s_m[wave][n16] = m[rt], s_l[wave][n16] = l[rt];
    if (n16 < left) {
#pragma unroll
      for (int d = 0; d < DT; ++d) {
        float4_t v = acc[rt][d];
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = B8 ? ldexpf(v[i], E - (int)X::SHIFT) : X::SHIFT != 0.f ? v[i] * exp2f(-X::SHIFT) : v[i];
        *(float4_t*)&s_acc[wave][n16][d * 16 + quad * 4] = v;
      }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < left * (HD / 4); i += PA_NW * 64) {
      const int r = i / (HD / 4), d = (i - r * (HD / 4)) * 4;
      float to = -INFINITY;
#pragma unroll
      for (int w = 0; w < PA_NW; ++w) to = fmaxf(to, s_m[w][r]);
      const float off = to == -INFINITY ? 0.f : to;
      float total = 0.f;
      float4_t o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int w = 0; w < PA_NW; ++w) {
        const float f = __builtin_amdgcn_exp2f(s_m[w][r] - off);
        // (a wave without keys has no sum, and its zeros take part in none that a NaN maximum would spoil)
        total += f * s_l[w][r];
        const float4_t v = *(const float4_t*)&s_acc[w][r][d];
#pragma unroll
        for (int k = 0; k < 4; ++k) o[k] += f * v[k];
      }
      const int rho = rho0 + rt * 16 + r, t = rho / group, head = h * group + rho - t * group;
      const int64_t row = (int64_t)row0 + t;
      if (a.splits > 1) {
        float* to_ = a.partial + ((row * a.heads + head) * a.splits + split) * (HD + 4);
        *(float4_t*)(to_ + d) = o;
        if (d == 0) to_[HD] = to, to_[HD + 1] = total;
      } else {
        const float inv = total > 0.f || total != total ? 1.f / total : 0.f;
        uint16_t w[4];
#pragma unroll
        for (int k = 0; k < 4; ++k)
          w[k] = a.bf16 ? __builtin_bit_cast(uint16_t, (bf16_t)(o[k] * inv)) : __builtin_bit_cast(uint16_t, (half_t)(o[k] * inv));
        const int64_t at = a.out_mb > 0 ? packed_act_offset((int)row, head * HD + d, a.out_mb) : row * a.ldo + head * HD + d;
        *(pg_u2*)((uint16_t*)a.out + at) = pg_u2{(uint32_t)w[0] | (uint32_t)w[1] << 16, (uint32_t)w[2] | (uint32_t)w[3] << 16};
      }
    }
  }
}

template <int F, int HD>
void pa_launch_rows(const PagedAttention& a, int rt, hipStream_t stream) {
  const dim3 grid((unsigned)((int64_t)a.nseq * a.row_blocks), (unsigned)a.kv_heads, (unsigned)a.splits);
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

}  // namespace
