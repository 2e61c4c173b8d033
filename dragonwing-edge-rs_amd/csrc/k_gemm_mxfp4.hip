// Products of rows (f16 or MXFP4) and MXFP4 weights: C = act(A W^T + bias).
//
// Both operands in MXFP4 are multiplied as they are: the scaled matrix
// instruction takes 16 rows x 128 elements of 4 bits a side, a lane's operand
// being one block of 32 (16 bytes) and its scale byte.
//
// f16 rows are multiplied as f16, and the weights widened to it: a value
// times its factor is an f16 value for factors of 2^-23 to 2^13, that is for
// any weights met in earnest.  Each wave looks at its scale bytes as it goes,
// and where one is outside that range (and its block not all zeros) it
// computes its part again in a form that holds for every factor: a quarter of
// the weights as bf16, four times each f16 element as the sum of two bf16 ones,
// so that every product is exact there too.  The quarter is what lets bf16 hold
// all of them: 6 x 2^127 is beyond its largest number, and 0.5 x 2^-127 / 4 is
// one of its subnormal numbers, which the matrix instruction takes as they are.
#include <algorithm>

#include "dw_common.h"
#include "mxfp4.h"

namespace dw {

namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef int i32x8 __attribute__((ext_vector_type(8)));

// Bias of four neighbours from column n on, 0 behind the row's end.
__device__ __forceinline__ f32x4 bias4(const GemmMxArgs& a, int n) {
  f32x4 b = {};
  if (!a.bias) return b;
#pragma unroll
  for (int r = 0; r < 4; ++r)
    if (n + r < a.n) b[r] = a.c_half ? h2f_ieee(((const uint16_t*)a.bias)[n + r]) : ((const float*)a.bias)[n + r];
  return b;
}

// e^-s is 2^(hi + lo), hi + lo = -s log2(e) to 2^-48 of it: exp2 and the
// reciprocal leave 2^-22 of the result, below an f16 C's 2^-11 and near the
// sum's own error in an f32 one.  1,209 x 7,712 x 832: MXFP4 rows 28.5 us, 33.4
// us with expf and a division, which leave 2^-24, and 23.6 us without SiLU; f16
// rows 39.4, 44.3 and 34.5 us.
__device__ __forceinline__ float silu(float s) {
  const float hi = s * -1.44269504f, lo = fmaf(s, -1.44269504f, -hi) + s * -1.92596300e-8f;
  const float e = __builtin_amdgcn_exp2f(hi);
  // an infinite e, or one of 0, has no use for lo, which an infinite s makes NaN
  const float d = 1.0f + (e > 0.0f && e < 3.0e38f ? fmaf(e * 0.693147181f, lo, e) : e);
  return 0.25f * s * __builtin_amdgcn_rcpf(0.25f * d);  // a reciprocal under 2^-126 would be 0
}

// Four neighbours of a row of C, from column n on: bias, activation and the
// one rounding of a sum.
__device__ __forceinline__ void store4(const GemmMxArgs& a, size_t row, int n, f32x4 s, f32x4 bias) {
  if (n >= a.n) return;
  const size_t at = row * a.n + n;
  s += bias;
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    if (a.act == ACT_RELU) s[r] = s[r] < 0.0f ? 0.0f : s[r];  // a NaN stays
    if (a.act == ACT_SILU) s[r] = silu(s[r]);
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

constexpr int kFewRows = 32;

// --- a few rows -----------------------------------------------------------------

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

template <bool MX, int MT, int NT, bool FEW>
__global__ __launch_bounds__(MT* NT == 1 ? 1024 : 512) void gemm_mx_rows_kernel(GemmMxArgs a) {
  extern __shared__ __align__(16) f32x4 sums[];  // [waves][NT * MT][64]
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
  const int n0 = blockIdx.x * 16 * NT, steps = ((a.k + 31) / 32 + 3) / 4;
  f32x4 acc[NT][MT];
  // the waves' shares are whole groups of four steps
  const int groups = (steps + 3) / 4;
  const int from = groups * wave / waves * 4, to = min(steps, groups * (wave + 1) / waves * 4);
  const Rows<MX, MT, NT, FEW> r(a, n0, (uint8_t*)sums + wave * 4 * Rows<MX, MT, NT, FEW>::kFewLine);
  const uint32_t odd = r.template sum<false>(from, to, acc);
  if constexpr (!MX)
    if (__ballot(odd != 0)) r.template sum<true>(from, to, acc);
  if (waves > 1) {
    if (FEW) __syncthreads();  // the rows' place becomes the sums'
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int u = 0; u < MT; ++u) sums[(wave * NT * MT + t * MT + u) * 64 + lane] = acc[t][u];
    __syncthreads();
  }
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int u = 0; u < MT; ++u) {
      if ((t * MT + u) % waves != wave) continue;
      f32x4 s = acc[t][u];
      if (waves > 1) {
        s = sums[(t * MT + u) * 64 + lane];
        for (int i = 1; i < waves; ++i) s += sums[(i * NT * MT + t * MT + u) * 64 + lane];
      }
      const int m = u * 16 + (lane & 15);
      const int n = n0 + t * 16 + (lane >> 4) * 4;
      if (m < a.m) store4(a, m, n, s, bias4(a, n));
    }
}

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

__global__ __launch_bounds__(256) void pad_kernel(Pads p) {
  const bool one = blockIdx.x < p.first;
  const unsigned groups = one ? p.first : gridDim.x - p.first;
  const size_t from = (size_t)(one ? blockIdx.x : blockIdx.x - p.first) * 256 + threadIdx.x, step = (size_t)groups * 256;
  if (one && p.x) {
    const unsigned pieces = p.lda / 8;
    for (size_t i = from; i < (size_t)p.m * pieces; i += step) {
      const size_t r = i / pieces;
      const int j = (int)(i - r * pieces) * 8;
      const uint16_t* x = p.x + r * p.k + j;
      Loose<uint16_t, 8> v;
      if (j + 8 <= p.k) {
        v = load_loose<uint16_t, 8>(x);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) v.v[e] = j + e < p.k ? x[e] : (uint16_t)0;
      }
      *(Loose<uint16_t, 8>*)__builtin_assume_aligned(p.x_to + i * 8, 16) = v;
    }
    return;
  }
  const uint8_t* s = one ? p.s[0] : p.s[1];
  uint32_t* to = one ? p.s_to[0] : p.s_to[1];
  const size_t rows = one ? p.rows[0] : p.rows[1];
  for (size_t i = from; i < rows * p.words; i += step) {
    const size_t r = i / (unsigned)p.words;
    const int b = (int)(i - r * p.words) * 4;
    uint32_t v = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) v |= (b + j < p.blocks ? (uint32_t)s[r * p.blocks + b + j] : 127u) << (8 * j);
    to[i] = v;
  }
}

template <bool MX, int MT, int NT, bool FEW = false>
void launch_rows(hipStream_t st, const GemmMxArgs& a) {
  const int tiles = (a.n + 16 * NT - 1) / (16 * NT), groups = ((a.k + 31) / 32 + 15) / 16;
  int waves = 1;
  while (waves < (MT * NT == 1 ? 16 : 8) && waves < groups && tiles * waves < 4096) waves *= 2;
  size_t lds = waves > 1 ? (size_t)waves * NT * MT * 1024 : 0;
  if (FEW) lds = std::max(lds, (size_t)waves * 4 * Rows<MX, MT, NT, FEW>::kFewLine);
  hipLaunchKernelGGL((gemm_mx_rows_kernel<MX, MT, NT, FEW>), dim3((unsigned)tiles), dim3(64u * waves), lds, st, a);
}

// Two tiles of 16 weight rows a wave halve what is read of A, where enough
// waves are left (16 f16 rows x 5120 x 5120: 10.9 us, 15.8 us with one tile;
// x 4096 x 14336: 22.6 us, 19.7 us with one; 24 x 4096 x 4096: 11.1 us, 9.4 us
// with one).  Up to four f16 rows come through LDS (one row x 4096 x 14336: 8.8
// us, 9.9 us without).
void rows(hipStream_t st, const GemmMxArgs& a) {
  const bool wide = a.n >= 5120;
  if (a.m > 16)
    if (wide) a.as ? launch_rows<true, 2, 2>(st, a) : launch_rows<false, 2, 2>(st, a);
    else a.as ? launch_rows<true, 2, 1>(st, a) : launch_rows<false, 2, 1>(st, a);
  else if (a.as)
    wide ? launch_rows<true, 1, 2>(st, a) : launch_rows<true, 1, 1>(st, a);
  else if (a.m <= 4)
    launch_rows<false, 1, 1, true>(st, a);
  else
    wide ? launch_rows<false, 1, 2>(st, a) : launch_rows<false, 1, 1>(st, a);
}

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
template <bool MX, int WM, int WN, int TM, int TN>
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
  uint32_t at_a[kLoadsA], at_w[kLoadsW], at_s[kLoadsS];  // a lane's pieces of the first stage, from the tile's rows
  const uint8_t *base_a, *base_w;

  // LDS keeps rows of A (and, for MXFP4 rows, of W) as they are, but the pieces
  // of row r stand at their index xor r: eight lanes that read one piece of
  // eight rows meet all banks.  Rows of W of 32 bytes stand 32 together, piece
  // by piece.
  __device__ __forceinline__ Tile(const GemmMxArgs& args, uint8_t* shared, int row0, int col0)
      : g(args), lds(shared), m0(row0), n0(col0) {
    wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    lane = threadIdx.x & 63, col = lane & 15, quad = lane >> 4, wm = wave % WM, wn = wave / WM;
    const size_t blocks = (g.k + 31) / 32;
    const size_t row_a = MX ? blocks * 16 : (size_t)g.lda * 2, row_w = blocks * 16;
    base_a = (const uint8_t*)g.a + m0 * row_a;
    base_w = g.w + n0 * row_w;
#pragma unroll
    for (int i = 0; i < kLoadsA; ++i) {
      const int r = (wave * kLoadsA + i) * (1024 / kLineA) + lane / (kLineA / 16);
      at_a[i] = (uint32_t)(min(r, g.m - 1 - m0) * row_a) + piece_a(i) * 16;  // rows behind the end are not stored
    }
#pragma unroll
    for (int i = 0; i < kLoadsW; ++i) {
      const int r = MX ? (wave * kLoadsW + i) * 8 + lane / 8 : (wave * kLoadsW + i) * 32 + lane % 32;
      at_w[i] = (uint32_t)(min(r, g.n - 1 - n0) * row_w) + piece_w() * 16;
    }
#pragma unroll
    for (int i = 0; i < kLoadsS; ++i) {
      const int r = scale_row(i);
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
      const uint8_t* p = pa + at_a[i];
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
    if constexpr (MORE != 0) {
      if (s % kSpan == 0) load_scales(next_scales, s / kSpan + 1);
      load<MORE == 1>(next, s + 1);
    }
    if constexpr (!kAhead) {
#pragma unroll
      for (int i = 0; i < kParts; ++i) {
        read(cur, scales, s, i, one);
        products<EXACT>(one, i, far, acc);
      }
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
    load_scales(lds + 2 * kStage, from / kSpan);
    load<true>(lds, from);
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
      if (g.ws[r * g.pitch + b] - 104u > 36u) {
        const uint4 q = *(const uint4*)(g.w + (r * blocks + b) * 16);
        odd |= ((q.x | q.y | q.z | q.w) & 0x77777777u) != 0;
      }
    }
    return odd;
  }
};

template <bool MX, int WM, int WN, int TM, int TN>
__global__ __launch_bounds__(WM* WN * 64) void gemm_mx_tile_kernel(GemmMxArgs a, int tiles_m, int tiles_n) {
  using T = Tile<MX, WM, WN, TM, TN>;
  extern __shared__ __align__(16) uint8_t lds[];
  // Neighbouring workgroups go to the 8 XCDs in turn: each takes a run of
  // tiles, eight rows of tiles wide, that share operands in its L2.
  const int total = tiles_m * tiles_n, id = blockIdx.x;
  const int per = total / 8, rest = total % 8, xcd = id % 8;
  const int tile = xcd * per + min(xcd, rest) + id / 8;
  constexpr int kBand = 8;
  const int band = tile / (kBand * tiles_n), high = min(kBand, tiles_m - band * kBand);
  const int in = tile - band * kBand * tiles_n;
  const int m0 = (band * kBand + in % high) * T::kRowsA, n0 = in / high * T::kRowsW;
  const int stages = (a.k + T::kDepth - 1) / T::kDepth, spans = (stages + T::kSpan - 1) / T::kSpan;
  const int from = (int)((long long)spans * blockIdx.y / gridDim.y) * T::kSpan;
  const int to = min(stages, (int)((long long)spans * (blockIdx.y + 1) / gridDim.y) * T::kSpan);
  f32x4 acc[TN][TM];
  const T t(a, lds, m0, n0);
  const uint32_t far = t.template sum<false>(from, to, acc);
  if constexpr (!MX) {
    if (__syncthreads_or(far != 0) && __syncthreads_or(t.outside(from, to))) t.template sum<true>(from, to, acc);
  }
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int m1 = m0 + wave % WM * TM * 16 + (lane & 15), n1 = n0 + wave / WM * TN * 16 + (lane >> 4) * 4;
  if (gridDim.y == 1) {
    // A row's columns go one after the other, so that its lines fill at once: 4,096
    // x 8,192 x 8,192 MXFP4 152 us, 185 us with a column's rows in turn.
    f32x4 bias[TN];
#pragma unroll
    for (int i = 0; i < TN; ++i) bias[i] = bias4(a, n1 + i * 16);
#pragma unroll
    for (int u = 0; u < TM; ++u) {
      if (m1 + u * 16 >= a.m) continue;
#pragma unroll
      for (int i = 0; i < TN; ++i) store4(a, m1 + u * 16, n1 + i * 16, acc[i][u], bias[i]);
    }
    return;
  }
  // a share of K: f32 sums, to be joined
  float* out = a.parts + (size_t)blockIdx.y * a.m * a.ldp;
#pragma unroll
  for (int u = 0; u < TM; ++u) {
    if (m1 + u * 16 >= a.m) continue;
#pragma unroll
    for (int i = 0; i < TN; ++i)
      if (n1 + i * 16 < a.ldp) *(f32x4*)(out + (size_t)(m1 + u * 16) * a.ldp + n1 + i * 16) = acc[i][u];
  }
}

// The shares' sums, in order, then bias, activation and rounding.
__global__ __launch_bounds__(256) void gemm_mx_join_kernel(GemmMxArgs a, int shares) {
  const int n = (blockIdx.x * 256 + threadIdx.x) * 4;
  if (n >= a.n) return;
  const f32x4 bias = bias4(a, n);
  for (int m = blockIdx.y; m < a.m; m += gridDim.y) {
    const float* p = a.parts + (size_t)m * a.ldp + n;
    f32x4 s = *(const f32x4*)p;
    for (int i = 1; i < shares; ++i) s += *(const f32x4*)(p + (size_t)i * a.m * a.ldp);
    store4(a, m, n, s, bias);
  }
}

}  // namespace

namespace {

// How a product is cut, and where its workspace lies.
struct Plan {
  bool big;      // tiles of 256 columns, else of 128
  int shares;    // of K
  size_t rows, scales_a, scales_w, parts, bytes;
};
Plan plan(const GemmMxArgs& a) {
  Plan p{};
  auto take = [&](size_t bytes) {
    const size_t at = p.bytes;
    p.bytes += (bytes + 255) / 256 * 256;
    return at;
  };
  const size_t blocks = (a.k + 31) / 32, pitch = (blocks + 15) / 16 * 16;
  if (!a.as && a.k % 8) p.rows = take((size_t)a.m * ((a.k + 7) / 8 * 8) * 2);
  if (a.m <= kFewRows) return p;
  if (blocks % 16) {
    if (a.as) p.scales_a = take(a.m * pitch);
    p.scales_w = take(a.n * pitch);
  }
  // The expected time of each tile and number of shares: rounds of workgroups
  // over the chip, each its stages and a start, and the joining of the shares
  // at 4 bytes a sum and share.  Measured stages of 256 x 256: f16 rows 1.45 us
  // on a few CUs, 1.83 us on all, MXFP4 rows 2.7 us; of 128 x 128, with one
  // workgroup a CU and with two: f16 rows 0.62 and 1.10 us, MXFP4 rows 1.0 and
  // 1.55 us.
  const int depth = a.as ? 256 : 64, spans = (a.k + 511) / 512;
  double best = 1e30;
  for (int big = 0; big < 2; ++big) {
    const int rows = big ? 256 : 128, cols = rows, slots = big ? 256 : 512;
    const size_t tiles = (size_t)((a.m + rows - 1) / rows) * ((a.n + cols - 1) / cols);
    for (int shares = 1; shares <= 64 && shares <= spans; shares *= 2) {
      const double rounds = (double)((tiles * shares + slots - 1) / slots);
      const double one = std::min(tiles * shares / 256.0, 1.0);                         // share of CUs that have one
      const double two = std::min(std::max(tiles * shares / 256.0 - 1.0, 0.0), 1.0);  // and that have two
      const double stage = a.as ? (big ? 2.7 : 1.0 + 0.55 * two) : (big ? 1.45 + 0.38 * one : 0.62 + 0.48 * two);
      double t = rounds * (3.0 + stage * ((spans + shares - 1) / shares * (512 / depth)));
      if (shares > 1) t += 2.0 + (double)a.m * a.n * 4 * (2 * shares + 1) / 8e6;
      if (t < best) best = t, p.big = big, p.shares = shares;
    }
  }
  if (p.shares > 1) p.parts = take((size_t)p.shares * a.m * ((a.n + 3) / 4 * 4) * 4);
  return p;
}

template <bool MX, int WM, int WN, int TM, int TN>
void launch_tiles(hipStream_t st, const GemmMxArgs& a, int shares) {
  using T = Tile<MX, WM, WN, TM, TN>;
  const int tm = (a.m + T::kRowsA - 1) / T::kRowsA, tn = (a.n + T::kRowsW - 1) / T::kRowsW;
  auto* k = gemm_mx_tile_kernel<MX, WM, WN, TM, TN>;
  hipLaunchKernelGGL(k, dim3((unsigned)((size_t)tm * tn), (unsigned)shares), dim3(WM * WN * 64), T::kLds, st, a, tm, tn);
}

}  // namespace

size_t gemm_mx_space(const GemmMxArgs& a) { return plan(a).bytes; }

void launch_gemm_mx(hipStream_t st, GemmMxArgs a, void* space) {
  const Plan p = plan(a);
  char* base = (char*)space;
  const int blocks = (a.k + 31) / 32, words = (blocks + 15) / 16 * 4;
  a.lda = (a.k + 7) / 8 * 8;
  a.pitch = words * 4;
  Pads pads{};
  pads.m = a.m, pads.k = a.k, pads.lda = a.lda, pads.blocks = blocks, pads.words = words;
  auto groups = [](size_t units) { return (unsigned)std::min<size_t>((units + 255) / 256, 4096); };
  unsigned others = 0;
  if (!a.as && a.k % 8) {
    pads.x = (const uint16_t*)a.a;
    a.a = pads.x_to = (uint16_t*)(base + p.rows);
    pads.first = groups((size_t)a.m * (a.lda / 8));
  }
  if (a.m > kFewRows && blocks % 16) {
    if (a.as) {
      pads.s[0] = a.as, pads.rows[0] = a.m;
      a.as = (const uint8_t*)(pads.s_to[0] = (uint32_t*)(base + p.scales_a));
      pads.first = groups((size_t)a.m * words);
    }
    pads.s[1] = a.ws, pads.rows[1] = a.n;
    a.ws = (const uint8_t*)(pads.s_to[1] = (uint32_t*)(base + p.scales_w));
    others = groups((size_t)a.n * words);
  }
  if (pads.first + others) hipLaunchKernelGGL(pad_kernel, dim3(pads.first + others), dim3(256), 0, st, pads);
  if (a.m <= kFewRows) {
    rows(st, a);
    DW_HIP(hipGetLastError());
    return;
  }
  a.parts = (float*)(base + p.parts);
  a.ldp = (a.n + 3) / 4 * 4;
  if (a.as)
    p.big ? launch_tiles<true, 2, 4, 8, 4>(st, a, p.shares) : launch_tiles<true, 2, 2, 4, 4>(st, a, p.shares);
  else
    p.big ? launch_tiles<false, 2, 4, 8, 4>(st, a, p.shares) : launch_tiles<false, 2, 2, 4, 4>(st, a, p.shares);
  if (p.shares > 1)
    hipLaunchKernelGGL(gemm_mx_join_kernel, dim3((unsigned)((a.n + 1023) / 1024), (unsigned)std::min(a.m, 65535)),
                       dim3(256), 0, st, a, p.shares);
  DW_HIP(hipGetLastError());
}

}  // namespace dw
