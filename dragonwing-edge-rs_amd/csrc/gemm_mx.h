// What the products with MXFP4 weights share (k_gemm_mxfp4.hip, one product of
// all rows; k_gemm_experts.hip, rows of many experts): a wave's part of a few
// rows, and tiles through LDS.
#pragma once

#include <type_traits>

#include "dw_common.h"
#include "expert_lists.h"
#include "mxfp4.h"

namespace dw {

// What is laid out anew before a product: f16 rows of A at a stride of whole 16
// bytes, zeros behind their ends; scale bytes with each row at a stride of 16
// bytes or more, 127 behind its end.  One launch: its first workgroups do one,
// the others the other.
struct Pads {
  const uint16_t* x;  // rows [m][k], or null
  uint16_t* x_to;     // [m][lda]
  const uint8_t* s[2];  // scales [rows][blocks], or null
  uint32_t* s_to[2];    // [rows][words]
  size_t rows[2];
  int m, k, lda, blocks, words;
  unsigned first;  // workgroups of x and s[0]; those behind them have s[1]
};
// `others`: workgroups of s[1].
void launch_pads(hipStream_t st, const Pads& p, unsigned others);

namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef int i32x8 __attribute__((ext_vector_type(8)));

// e^-s is 2^(hi + lo), hi + lo = -s log2(e) to 2^-48 of it: exp2 and the
// reciprocal leave 2^-22 of the result, below an f16 C's 2^-11 and near the
// sum's own error in an f32 one; where e is beyond f32 the result, under 2^-121,
// is 0.  1,209 x 7,712 x 832: MXFP4 rows 28.5 us, 33.4 us with expf and a
// division, which leave 2^-24, and 23.6 us without SiLU; f16 rows 39.4, 44.3 and
// 34.5 us.
__device__ __forceinline__ float silu(float s) {
  const float hi = s * -1.44269504f, lo = fmaf(s, -1.44269504f, -hi) + s * -1.92596300e-8f;
  const float e = __builtin_amdgcn_exp2f(hi);
  // an infinite e, or one of 0, has no use for lo, which an infinite s makes NaN
  const float d = 1.0f + (e > 0.0f && e < 3.0e38f ? fmaf(e * 0.693147181f, lo, e) : e);
  return 0.25f * s * __builtin_amdgcn_rcpf(0.25f * d);  // a reciprocal under 2^-126 would be 0
}

// The same for a result of f16: its exponent's rounding (|s| 2^-24) stands in e as it
// is, 2^-17 of a value at most, where half a step of f16 is 2^-11.  Half the
// instructions, which at a tile's end nothing hides.
__device__ __forceinline__ float silu_f16(float s) {
  const float e = __builtin_amdgcn_exp2f(s * -1.44269504f);
  return 0.25f * s * __builtin_amdgcn_rcpf(fmaf(e, 0.25f, 0.25f));
}

// Bias of four neighbours from column n on, 0 behind the row's end.
__device__ __forceinline__ f32x4 bias4(const GemmMxArgs& a, int n) {
  f32x4 b = {};
  if (!a.bias) return b;
#pragma unroll
  for (int r = 0; r < 4; ++r)
    if (n + r < a.n) b[r] = a.c_half ? h2f_ieee(((const uint16_t*)a.bias)[n + r]) : ((const float*)a.bias)[n + r];
  return b;
}

// Four neighbours of a row of C, from column n on: bias, activation and the
// one rounding of a sum.  GATED: the activation may be the gated one, whose
// neighbours two by two make one column of C.
template <bool GATED = false>
__device__ __forceinline__ void store4(const GemmMxArgs& a, size_t row, int n, f32x4 s, f32x4 bias) {
  if (n >= a.n) return;
  const size_t at = row * a.n + n;
  s += bias;
  const bool quick = GATED && a.c_half;
  if (GATED && a.act == ACT_SWIGLU) {  // n and a.n are even
    const float y[2] = {(quick ? silu_f16(s[0]) : silu(s[0])) * s[1], (quick ? silu_f16(s[2]) : silu(s[2])) * s[3]};
    if (n + 4 <= a.n) {
      if (a.c_half)
        store_loose<uint16_t, 2>((uint16_t*)a.c + at / 2, {narrow<uint16_t>(y[0]), narrow<uint16_t>(y[1])});
      else
        store_loose<float, 2>((float*)a.c + at / 2, {y[0], y[1]});
    } else if (a.c_half) {
      ((uint16_t*)a.c)[at / 2] = narrow<uint16_t>(y[0]);
    } else {
      ((float*)a.c)[at / 2] = y[0];
    }
    return;
  }
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    if (a.act == ACT_RELU) s[r] = s[r] < 0.0f ? 0.0f : s[r];  // a NaN stays
    if (a.act == ACT_SILU) s[r] = quick ? silu_f16(s[r]) : silu(s[r]);
  }
  if (n + 4 <= a.n) {
    if (a.c_half) {
      Loose<uint16_t, 4> h;
#pragma unroll
      for (int r = 0; r < 4; ++r) h.v[r] = narrow<uint16_t>(s[r]);
      store_loose<uint16_t, 4>((uint16_t*)a.c + at, h);
    } else {
      Loose<float, 4> h;
#pragma unroll
      for (int r = 0; r < 4; ++r) h.v[r] = s[r];
      store_loose<float, 4>((float*)a.c + at, h);
    }
    return;
  }
#pragma unroll
  for (int r = 0; r < 4; ++r)
    if (n + r < a.n) {
      if (a.c_half)
        ((uint16_t*)a.c)[at + r] = narrow<uint16_t>(s[r]);
      else
        ((float*)a.c)[at + r] = s[r];
    }
}

// Sixteen scale bytes from block b of a row of `blocks`: four steps of four
// blocks.  Bytes behind the row's end are 127, the factor one.
__device__ __forceinline__ uint4 scales16(const uint8_t* row, int b, int blocks) {
  uint4 v;
  if (b + 16 <= blocks) {
    __builtin_memcpy(&v, row + b, 16);
  } else {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      w[i] = 0;
#pragma unroll
      for (int j = 0; j < 4; ++j) w[i] |= (b + i * 4 + j < blocks ? (uint32_t)row[b + i * 4 + j] : 127u) << (8 * j);
    }
    v = make_uint4(w[0], w[1], w[2], w[3]);
  }
  return v;
}
__device__ __forceinline__ uint32_t word(const uint4& v, int i) { return i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w; }

template <int J>
__device__ __forceinline__ h16x2 pair_f16(uint32_t w, float s) {
  return __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, s, J);
}
__device__ __forceinline__ f16x8 eight_f16(uint32_t w, float s) {
  const h16x2 a = pair_f16<0>(w, s), b = pair_f16<1>(w, s), c = pair_f16<2>(w, s), d = pair_f16<3>(w, s);
  return f16x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}
template <int J>
__device__ __forceinline__ uint32_t pair_bf16(uint32_t w, float s) {
  return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, J));
}
// A quarter of eight weights; `s` has their scale byte in bits 30:23.
__device__ __forceinline__ bf16x8 quarters_bf16(uint32_t w, float s) {
  const uint32_t byte = __builtin_bit_cast(uint32_t, s) >> 23 & 255u;
  const float f = mx_scale(byte == 255u ? 255u : max(byte, 2u) - 2u);
  uint32_t h[4] = {pair_bf16<0>(w, f), pair_bf16<1>(w, f), pair_bf16<2>(w, f), pair_bf16<3>(w, f)};
  if (__ballot(byte < 2u)) {  // factors of 2^-129 and 2^-128, which no scale byte stands for
    const float rest = byte == 0u ? 0.25f : byte == 1u ? 0.5f : 1.0f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float lo = __builtin_bit_cast(float, h[i] << 16) * rest, hi = __builtin_bit_cast(float, h[i] & 0xFFFF0000u) * rest;
      h[i] = __builtin_bit_cast(uint32_t, lo) >> 16 | (__builtin_bit_cast(uint32_t, hi) & 0xFFFF0000u);
    }
  }
  return __builtin_bit_cast(bf16x8, make_uint4(h[0], h[1], h[2], h[3]));
}
// Four times f16 elements as bf16 ones whose sum they are: the upper eight bits
// of the significand, and what is left (nothing, for an infinity).  Both are
// bf16 values, the upper halves of their f32 forms.
__device__ __forceinline__ void halves(f16x8 x, bf16x8* hi, bf16x8* lo) {
  const uint4 words = __builtin_bit_cast(uint4, x);
  uint32_t h[4], l[4];
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const uint16_t b = (uint16_t)(word(words, e / 2) >> (16 * (e & 1)));
    const bool odd = (b & 0x7C00u) == 0x7C00u;  // infinities and NaN
    const float top = 4.0f * h2f_ieee(odd ? b : (uint16_t)(b & 0xFFF8u));
    const uint32_t t = __builtin_bit_cast(uint32_t, top);
    const uint32_t r = odd ? 0u : __builtin_bit_cast(uint32_t, fmaf(h2f_ieee(b), 4.0f, -top));
    h[e / 2] = e % 2 ? h[e / 2] | (t & 0xFFFF0000u) : t >> 16;
    l[e / 2] = e % 2 ? l[e / 2] | (r & 0xFFFF0000u) : r >> 16;
  }
  *hi = __builtin_bit_cast(bf16x8, make_uint4(h[0], h[1], h[2], h[3]));
  *lo = __builtin_bit_cast(bf16x8, make_uint4(l[0], l[1], l[2], l[3]));
}
__device__ __forceinline__ f32x4 times_exact(bf16x8 v, f16x8 x, f32x4 acc) {
  bf16x8 hi, lo;
  halves(x, &hi, &lo);
  acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(v, hi, acc, 0, 0, 0);
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(v, lo, acc, 0, 0, 0);
}

// Rows that fit 16 x MT columns of the matrix instruction, whose rows are the
// weights': NT tiles of 16 of them a workgroup, K shared by its waves, whose
// sums meet in LDS in order.
//
// Bound by the weights' bytes: 17/32 of one an element, read once.  A lane's
// operand is a whole block, four lanes side by side read 64 bytes of a row,
// and four steps' loads are in flight at a time; each workgroup reads the
// rows of A again from L2, which NT divides.  One f16 row x 14336 x 4096:
// 10.1 us a call among others (3.1 TB/s); 16 MXFP4 rows x 8192 x 8192: 9.8 us
// (3.7 TB/s).
// FEW: f16 rows, at most four, that a wave brings to LDS whole, an element
// once: the matrix instruction's operand has 16 columns, and as loads of its
// own each would cost 64 bytes a lane and step.
template <bool MX, int MT, int NT, bool FEW>
struct Rows {
  const GemmMxArgs& g;
  const uint8_t *w[NT], *ws[NT], *x[MT], *xs[MT];
  int lane, col, quad, blocks;
  uint8_t* few;  // this wave's rows in LDS
  static constexpr int kFewLine = 1024 + 16;
  __device__ __forceinline__ Rows(const GemmMxArgs& args, int n0, uint8_t* lds) : g(args), few(lds) {
    lane = threadIdx.x & 63, col = lane & 15, quad = lane >> 4, blocks = (g.k + 31) / 32;
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const size_t n = min(n0 + t * 16 + col, g.n - 1);  // rows behind the end are not stored, on both sides
      w[t] = g.w + (n * blocks + quad) * 16;
      ws[t] = g.ws + n * blocks;
    }
#pragma unroll
    for (int u = 0; u < MT; ++u) {
      const size_t m = min(u * 16 + col, g.m - 1);
      x[u] = (const uint8_t*)g.a + (MX ? (m * blocks + quad) * 16 : (m * g.lda + quad * 32) * 2);
      xs[u] = MX ? g.as + m * blocks : nullptr;
    }
  }
  // Four steps from s0; ALL: none of them reaches behind the end of K.
  template <bool EXACT, bool ALL>
  __device__ __forceinline__ void four(int s0, int to, uint32_t* odd, f32x4 (&acc)[NT][MT]) const {
    uint4 wv[NT][4], sw[NT], sx[MT], xv[MT][MX ? 4 : 16];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        wv[t][i] = ALL || (s0 + i < to && (s0 + i) * 4 + quad < blocks) ? *(const uint4*)(w[t] + (size_t)(s0 + i) * 64)
                                                                        : make_uint4(0, 0, 0, 0);
      if constexpr (ALL)
        __builtin_memcpy(&sw[t], ws[t] + s0 * 4, 16);
      else
        sw[t] = scales16(ws[t], s0 * 4, blocks);
    }
#pragma unroll
    for (int u = 0; u < MT; ++u) {
      if constexpr (MX) {
        if constexpr (ALL)
          __builtin_memcpy(&sx[u], xs[u] + s0 * 4, 16);
        else
          sx[u] = scales16(xs[u], s0 * 4, blocks);
      }
      if constexpr (FEW) {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          if (r >= g.m) break;
          const int k = s0 * 128 + lane * 8;
          const uint4 v = ALL || (k < g.lda && s0 + lane / 16 < to)
                              ? *(const uint4*)((const uint8_t*)g.a + ((size_t)r * g.lda + k) * 2)
                              : make_uint4(0, 0, 0, 0);
          *(uint4*)(few + r * kFewLine + lane * 16) = v;
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
        const uint8_t* p = few + min(col, g.m - 1) * kFewLine + quad * 64;
#pragma unroll
        for (int i = 0; i < 16; ++i) xv[u][i] = *(const uint4*)(p + i / 4 * 256 + i % 4 * 16);
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
        continue;
      }
#pragma unroll
      for (int i = 0; i < (MX ? 4 : 16); ++i) {
        if constexpr (MX)
          xv[u][i] = ALL || (s0 + i < to && (s0 + i) * 4 + quad < blocks) ? *(const uint4*)(x[u] + (size_t)(s0 + i) * 64)
                                                                          : make_uint4(0, 0, 0, 0);
        else
          xv[u][i] = ALL || (s0 + i / 4 < to && ((s0 + i / 4) * 4 + quad) * 32 + i % 4 * 8 < g.lda)
                         ? *(const uint4*)(x[u] + (size_t)(s0 + i / 4) * 256 + i % 4 * 16)
                         : make_uint4(0, 0, 0, 0);
      }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        const uint32_t v = word(sw[t], i);
        if constexpr (MX) {
          const i32x8 p = {(int)wv[t][i].x, (int)wv[t][i].y, (int)wv[t][i].z, (int)wv[t][i].w, 0, 0, 0, 0};
#pragma unroll
          for (int u = 0; u < MT; ++u) {
            const i32x8 q = {(int)xv[u][i].x, (int)xv[u][i].y, (int)xv[u][i].z, (int)xv[u][i].w, 0, 0, 0, 0};
            acc[t][u] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(p, q, acc[t][u], 4, 4, 0, (int)(v >> (8 * quad)),
                                                                        0, (int)(word(sx[u], i) >> (8 * quad)));
          }
        } else {
          const uint32_t fb = __builtin_amdgcn_alignbit(v, v, 8 * quad + 9);  // byte `quad` to bits 30:23
          const float f = __builtin_bit_cast(float, fb);
          if constexpr (!EXACT) {
            const uint4 q = wv[t][i];
            const uint32_t some = (q.x | q.y | q.z | q.w) & 0x77777777u;
            *odd |= (fb & 0x7F800000u) - (104u << 23) > (36u << 23) ? some : 0u;
          }
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            if constexpr (EXACT) {
              const bf16x8 e = quarters_bf16(word(wv[t][i], j), f);
#pragma unroll
              for (int u = 0; u < MT; ++u)
                acc[t][u] = times_exact(e, __builtin_bit_cast(f16x8, xv[u][i * 4 + j]), acc[t][u]);
            } else {
              const f16x8 e = eight_f16(word(wv[t][i], j), f);
#pragma unroll
              for (int u = 0; u < MT; ++u)
                acc[t][u] = __builtin_amdgcn_mfma_f32_16x16x32_f16(e, __builtin_bit_cast(f16x8, xv[u][i * 4 + j]),
                                                                  acc[t][u], 0, 0, 0);
            }
          }
        }
      }
    }
  }
  template <bool EXACT>
  __device__ __forceinline__ uint32_t sum(int from, int to, f32x4 (&acc)[NT][MT]) const {
    uint32_t odd = 0;  // a factor that f16 does not hold
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int u = 0; u < MT; ++u) acc[t][u] = f32x4{};
    const int whole = min(to, MX ? blocks / 4 : g.lda / 128);
    int s = from;
    for (; s + 4 <= whole; s += 4) four<EXACT, true>(s, to, &odd, acc);
    for (; s < to; s += 4) four<EXACT, false>(s, to, &odd, acc);
    return odd;
  }
};
// --- many rows --------------------------------------------------------------------

// All of the wave's loads and LDS reads done, then all waves here.
__device__ __forceinline__ void settle() {
  __builtin_amdgcn_s_waitcnt(7 << 4);
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

__device__ __align__(16) const uint32_t kZeros[4] = {0, 0, 0, 0};

typedef __attribute__((address_space(3))) void* LdsPtr;

// A tile of WM x TM x 16 rows of A and WN x TN x 16 of W by WM x WN waves.
//
// K goes by in stages of whole cache lines: 256 elements of MXFP4 rows, 64 of
// f16 rows (128 bytes); of W 32 bytes a row there.  Loads write
// to LDS directly, a stage ahead, into the half of LDS that the last stage
// left; a stage's products come in parts of one matrix instruction's depth,
// each part's operands read ahead of the products of the part before, also
// over the end of a stage.  Scales come four bytes an operand row and 128
// elements: 16 bytes a row at a time, which last for 512 elements, because
// each such load touches a line for every row.
//
// 4,096 x 8,192 x 8,192: MXFP4 rows 152 us (3.6 PFLOP/s; 190 us in tiles of 128
// x 128); f16 rows 420 us (1.31 PFLOP/s; a library's product with f16 weights in
// the same layout reaches 1.58), bound by the conversions of the weights, which
// larger tiles share among more rows (128 x 128: 508 us).
//
// LIST: rows of A as a list has them, place m0 + i of it for row i of the tile
// (g.a and g.as from row 0 on; at most 2^32 pieces of 16 bytes), and scale rows
// of `blocks` bytes as they are, of any alignment.
template <bool MX, int WM, int WN, int TM, int TN, bool LIST = false>
struct Tile {
  static constexpr int kWaves = WM * WN, kRowsA = WM * TM * 16, kRowsW = WN * TN * 16;
  static constexpr int kDepth = MX ? 256 : 64, kParts = 2, kSpan = 512 / kDepth;
  static constexpr int kLineA = 128, kLineW = MX ? 128 : 32;  // bytes of a row and stage
  static constexpr int kA = kRowsA * kLineA, kW = kRowsW * kLineW, kStage = kA + kW;
  static constexpr int kScaleRows = (MX ? kRowsA : 0) + kRowsW, kScales = kScaleRows * 16;
  static constexpr int kLds = 2 * (kStage + kScales);
  static constexpr bool kAhead = TM * TN <= 16;  // the others' sums leave no registers for operands read ahead
  // a wave's loads of a stage, 64 pieces of 16 bytes each, and of scales
  static constexpr int kLoadsA = kA / 1024 / kWaves, kLoadsW = kW / 1024 / kWaves, kLoadsS = (kScaleRows / 64 + kWaves - 1) / kWaves;
  static_assert(kLoadsA * kWaves * 1024 == kA && kLoadsW * kWaves * 1024 == kW, "whole loads");

  const GemmMxArgs& g;
  uint8_t* lds;
  int m0, n0, wave, lane, col, quad, wm, wn;
  // a lane's pieces of the first stage, from the tile's rows (LIST: those of A in 16 bytes, from row 0)
  uint32_t at_a[kLoadsA], at_w[kLoadsW];
  typename std::conditional<LIST, size_t, uint32_t>::type at_s[kLoadsS];
  const uint8_t *base_a, *base_w;

  // LDS keeps rows of A (and, for MXFP4 rows, of W) as they are, but the pieces
  // of row r stand at their index xor r: eight lanes that read one piece of
  // eight rows meet all banks.  Rows of W of 32 bytes stand 32 together, piece
  // by piece.
  __device__ __forceinline__ Tile(const GemmMxArgs& args, uint8_t* shared, int row0, int col0, const RowList& list = {})
      : g(args), lds(shared), m0(row0), n0(col0) {
    wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    lane = threadIdx.x & 63, col = lane & 15, quad = lane >> 4, wm = wave % WM, wn = wave / WM;
    const size_t blocks = (g.k + 31) / 32;
    const size_t row_a = MX ? blocks * 16 : (size_t)g.lda * 2, row_w = blocks * 16;
    base_a = (const uint8_t*)g.a + (LIST ? 0 : m0 * row_a);
    base_w = g.w + n0 * row_w;
#pragma unroll
    for (int i = 0; i < kLoadsA; ++i) {
      const int r = (wave * kLoadsA + i) * (1024 / kLineA) + lane / (kLineA / 16);
      const int in = min(r, g.m - 1 - m0);  // rows behind the end are not stored
      at_a[i] = LIST ? list.row(m0 + in) * (uint32_t)(row_a / 16) + piece_a(i) : (uint32_t)(in * row_a) + piece_a(i) * 16;
    }
#pragma unroll
    for (int i = 0; i < kLoadsW; ++i) {
      const int r = MX ? (wave * kLoadsW + i) * 8 + lane / 8 : (wave * kLoadsW + i) * 32 + lane % 32;
      at_w[i] = (uint32_t)(min(r, g.n - 1 - n0) * row_w) + piece_w() * 16;
    }
#pragma unroll
    for (int i = 0; i < kLoadsS; ++i) {
      const int r = scale_row(i);
      if constexpr (LIST)
        at_s[i] = (MX && r < kRowsA ? (size_t)list.row(m0 + min(r, g.m - 1 - m0))
                                    : (size_t)min(r - (MX ? kRowsA : 0), g.n - 1 - n0)) * blocks;
      else
        at_s[i] = (uint32_t)((MX && r < kRowsA ? min(r, g.m - 1 - m0) : min(r - (MX ? kRowsA : 0), g.n - 1 - n0)) * g.pitch);
    }
  }
  __device__ __forceinline__ int piece_a(int i) const {
    const int r = i * (1024 / kLineA) + lane / (kLineA / 16);  // of the row's last three bits
    return lane % (kLineA / 16) ^ (r & 7);
  }
  __device__ __forceinline__ int piece_w() const { return MX ? lane % 8 ^ lane / 8 : lane / 32; }
  __device__ __forceinline__ int scale_row(int i) const { return (wave + i * kWaves) % (kScaleRows / 64) * 64 + lane; }

  // LAST: some of the stage's pieces may lie behind the end of K.
  template <bool LAST>
  __device__ __forceinline__ void load(uint8_t* __restrict__ slot, int stage) const {
    const uint8_t* pa = base_a + (size_t)stage * kLineA;
    const uint8_t* pw = base_w + (size_t)stage * kLineW;
    const int pieces = LAST ? (MX ? (g.k + 31) / 32 : g.lda / 8) - stage * 8 : 0;
    const int pieces_w = LAST ? (g.k + 31) / 32 - stage * (kDepth / 32) : 0;
#pragma unroll
    for (int i = 0; i < kLoadsA; ++i) {
      const uint8_t* p = LIST ? pa + (size_t)at_a[i] * 16 : pa + at_a[i];
      if (LAST && piece_a(i) >= pieces) p = (const uint8_t*)kZeros;
      __builtin_amdgcn_global_load_lds((const void*)p, (LdsPtr)(slot + (wave * kLoadsA + i) * 1024), 16, 0, 0);
    }
#pragma unroll
    for (int i = 0; i < kLoadsW; ++i) {
      const uint8_t* p = pw + at_w[i];
      if (LAST && piece_w() >= pieces_w) p = (const uint8_t*)kZeros;
      __builtin_amdgcn_global_load_lds((const void*)p, (LdsPtr)(slot + kA + (wave * kLoadsW + i) * 1024), 16, 0, 0);
    }
  }
  // LIST: the scales of 512 elements through registers
  // (loads to LDS want whole words); bytes behind a row's end are 127.
  struct Loose16 {
    uint4 v[kLoadsS];
  };
  __device__ __forceinline__ void fetch_scales(Loose16& r, int span) const {
    const int blocks = (g.k + 31) / 32, b = span * 16;
    if (b >= blocks) return;
#pragma unroll
    for (int i = 0; i < kLoadsS; ++i) {
      const bool of_a = MX && scale_row(i) < kRowsA;  // the same for the wave
      const uint8_t* p = (of_a ? g.as : g.ws + (size_t)n0 * blocks) + at_s[i];
      if (b + 16 <= blocks)
        __builtin_memcpy(&r.v[i], p + b, 16);
      else
        r.v[i] = scales16(p, b, blocks);
    }
  }
  __device__ __forceinline__ void place_scales(uint8_t* __restrict__ slot, const Loose16& r, int span) const {
    if (span * 16 >= (g.k + 31) / 32) return;
#pragma unroll
    for (int i = 0; i < kLoadsS; ++i) *(uint4*)(slot + scale_row(i) * 16) = r.v[i];
  }
  // The scales of 512 elements.
  __device__ __forceinline__ void load_scales(uint8_t* __restrict__ slot, int span) const {
    const int at = min(span, g.pitch / 16 - 1) * 16;
#pragma unroll
    for (int i = 0; i < kLoadsS; ++i) {
      const bool of_a = MX && scale_row(i) < kRowsA;  // the same for the wave
      const uint8_t* p = (of_a ? g.as + (size_t)m0 * g.pitch : g.ws + (size_t)n0 * g.pitch) + at + at_s[i];
      __builtin_amdgcn_global_load_lds((const void*)p, (LdsPtr)(slot + (wave + i * kWaves) % (kScaleRows / 64) * 1024), 16,
                                       0, 0);
    }
  }

  // A wave's operands of a part.
  struct Operands {
    uint4 x[TM];
    uint32_t fx[MX ? TM : 1];
    uint4 y[MX ? TN : 1];
    uint32_t word[MX ? 1 : TN], fw[TN];
  };
  __device__ __forceinline__ void read(const uint8_t* __restrict__ p, const uint8_t* __restrict__ scales, int stage,
                                       int part, Operands& r) const {
    const uint8_t* pa = p + wm * TM * 16 * kLineA + col * kLineA + (((quad ^ (col & 7)) ^ part * 4) * 16);
#pragma unroll
    for (int u = 0; u < TM; ++u) r.x[u] = *(const uint4*)(pa + u * 16 * kLineA);
    if constexpr (MX) {
      const uint8_t* sa = scales + (wm * TM * 16 + col) * 16 + (stage & 1) * 8 + part * 4 + quad;
      const uint8_t* sw = scales + (kRowsA + wn * TN * 16 + col) * 16 + (stage & 1) * 8 + part * 4 + quad;
      const uint8_t* pw = p + kA + wn * TN * 2048 + col * 128 + (((quad ^ (col & 7)) ^ part * 4) * 16);
#pragma unroll
      for (int u = 0; u < TM; ++u) r.fx[u] = sa[u * 256];
#pragma unroll
      for (int t = 0; t < TN; ++t) r.y[t] = *(const uint4*)(pw + t * 2048);
#pragma unroll
      for (int t = 0; t < TN; ++t) r.fw[t] = sw[t * 256];
    } else {
      const uint8_t* sw = scales + (wn * TN * 16 + col) * 16 + (stage & 7) * 2;
      const uint8_t* pw = p + kA + wn * TN * 512 + part * 512 + col * 16 + quad * 4;
#pragma unroll
      for (int t = 0; t < TN; ++t) r.word[t] = *(const uint32_t*)(pw + t / 2 * 1024 + t % 2 * 256);
#pragma unroll
      for (int t = 0; t < TN; ++t) r.fw[t] = *(const uint16_t*)(sw + t * 256);
    }
  }
  template <bool EXACT>
  static __device__ __forceinline__ void multiply(const Operands& r, int part, uint32_t* far, f32x4 (&acc)[TN][TM]) {
#pragma unroll
    for (int t = 0; t < TN; ++t) {
      if constexpr (MX) {
        const i32x8 q = {(int)r.y[t].x, (int)r.y[t].y, (int)r.y[t].z, (int)r.y[t].w, 0, 0, 0, 0};
#pragma unroll
        for (int u = 0; u < TM; ++u) {
          const i32x8 v = {(int)r.x[u].x, (int)r.x[u].y, (int)r.x[u].z, (int)r.x[u].w, 0, 0, 0, 0};
          acc[t][u] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(q, v, acc[t][u], 4, 4, 0, (int)r.fw[t], 0,
                                                                      (int)r.fx[u]);
        }
      } else {
        const float f = __builtin_bit_cast(float, r.fw[t] << (23 - 8 * part));
        if constexpr (EXACT) {
          const bf16x8 v = quarters_bf16(r.word[t], f);
#pragma unroll
          for (int u = 0; u < TM; ++u) acc[t][u] = times_exact(v, __builtin_bit_cast(f16x8, r.x[u]), acc[t][u]);
        } else {
          // factors of 2^-15 to 1, as weights have them, both parts' at a time
          if (part == 0) *far |= (r.fw[t] ^ 0x7070u) & 0xF0F0u;
          const f16x8 v = eight_f16(r.word[t], f);
#pragma unroll
          for (int u = 0; u < TM; ++u)
            acc[t][u] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, __builtin_bit_cast(f16x8, r.x[u]), acc[t][u], 0, 0, 0);
        }
      }
    }
  }

  // Reads stay ahead of the products, and the products of a wave that has its
  // operands go before the other waves' reads.
  template <bool EXACT>
  static __device__ __forceinline__ void products(const Operands& r, int part, uint32_t* far, f32x4 (&acc)[TN][TM]) {
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_setprio(1);
    multiply<EXACT>(r, part, far, acc);
    __builtin_amdgcn_s_setprio(0);
    __builtin_amdgcn_sched_barrier(0);
  }

  // Stages [from, to), from a multiple of kSpan.  A stage reads from `cur` and
  // loads into `next`: that the two are apart is what lets reads go ahead of
  // loads in flight (else each would wait for them).
  template <bool EXACT, int MORE>  // MORE: 0 no stage follows, 1 the last may, 2 any
  __device__ __forceinline__ void stage(const uint8_t* __restrict__ cur, const uint8_t* __restrict__ scales,
                                        uint8_t* __restrict__ next, uint8_t* __restrict__ next_scales, int s,
                                        Operands& one, Operands& two, uint32_t* far, f32x4 (&acc)[TN][TM]) const {
    Loose16 loose;
    const bool turn = MORE != 0 && s % kSpan == 0;
    if constexpr (MORE != 0) {
      if (turn) {
        if constexpr (LIST)
          fetch_scales(loose, s / kSpan + 1);
        else
          load_scales(next_scales, s / kSpan + 1);
      }
      load<MORE == 1>(next, s + 1);
    }
    auto placed = [&] {
      if constexpr (LIST && MORE != 0)
        if (turn) place_scales(next_scales, loose, s / kSpan + 1);
    };
    if constexpr (!kAhead) {
#pragma unroll
      for (int i = 0; i < kParts; ++i) {
        read(cur, scales, s, i, one);
        products<EXACT>(one, i, far, acc);
      }
      placed();
      return;
    }
    read(cur, scales, s, 0, one);
    products<EXACT>(two, kParts - 1, far, acc);  // of the stage before
#pragma unroll
    for (int i = 1; i < kParts; ++i) {
      Operands& now = i % 2 ? one : two;
      Operands& then = i % 2 ? two : one;
      read(cur, scales, s, i, then);
      products<EXACT>(now, i - 1, far, acc);
    }
    placed();
  }
  template <bool EXACT>
  __device__ __forceinline__ uint32_t sum(int from, int to, f32x4 (&acc)[TN][TM]) const {
    uint32_t far = 0;
#pragma unroll
    for (int t = 0; t < TN; ++t)
#pragma unroll
      for (int u = 0; u < TM; ++u) acc[t][u] = f32x4{};
    Operands one, two = {};  // zeros times zeros come before the first stage
    if constexpr (!MX) {
#pragma unroll
      for (int t = 0; t < TN; ++t) two.fw[t] = 0x7070u;
    }
    if constexpr (LIST) {
      Loose16 loose;
      fetch_scales(loose, from / kSpan);
      load<true>(lds, from);
      place_scales(lds + 2 * kStage, loose, from / kSpan);
    } else {
      load_scales(lds + 2 * kStage, from / kSpan);
      load<true>(lds, from);
    }
    auto slot = [&](int i) { return lds + ((i - from) & 1) * kStage; };
    auto scales = [&](int span) { return lds + 2 * kStage + ((span - from / kSpan) & 1) * kScales; };
    int s = from;
    for (; s < to - 2; ++s) {
      settle();
      stage<EXACT, 2>(slot(s), scales(s / kSpan), slot(s + 1), scales(s / kSpan + 1), s, one, two, &far, acc);
    }
    if (s < to - 1) {
      settle();
      stage<EXACT, 1>(slot(s), scales(s / kSpan), slot(s + 1), scales(s / kSpan + 1), s, one, two, &far, acc);
      ++s;
    }
    settle();
    stage<EXACT, 0>(slot(s), scales(s / kSpan), slot(s + 1), scales(s / kSpan + 1), s, one, two, &far, acc);
    if constexpr (kAhead) products<EXACT>(two, kParts - 1, &far, acc);
    settle();
    return far;
  }
  // Whether f16 does not hold a weight of the tile: factors one by one.
  __device__ __forceinline__ bool outside(int from, int to) const {
    const int blocks = (g.k + 31) / 32, b0 = from * (kDepth / 32), b1 = min(to * (kDepth / 32), blocks);
    bool odd = false;
    for (int i = threadIdx.x; i < (b1 - b0) * kRowsW; i += kWaves * 64) {
      const size_t r = min(n0 + i / (b1 - b0), g.n - 1), b = b0 + i % (b1 - b0);
      if (g.ws[r * (LIST ? blocks : g.pitch) + b] - 104u > 36u) {
        const uint4 q = *(const uint4*)(g.w + (r * blocks + b) * 16);
        odd |= ((q.x | q.y | q.z | q.w) & 0x77777777u) != 0;
      }
    }
    return odd;
  }
};

}  // namespace

}  // namespace dw
