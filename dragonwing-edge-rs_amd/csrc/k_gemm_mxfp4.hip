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
// computes its part again in a form that holds for every factor: weights as
// bf16 (exact from 2^-126 up), each f16 element as the sum of two bf16 ones,
// so that every product is exact there too.
#include <algorithm>

#include "dw_common.h"
#include "mxfp4.h"

namespace dw {

namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef int i32x8 __attribute__((ext_vector_type(8)));

// bias, activation and the one rounding of a sum
__device__ __forceinline__ float finish(const GemmMxArgs& a, int col, float s) {
  if (a.bias) s += a.c_half ? h2f_ieee(((const uint16_t*)a.bias)[col]) : ((const float*)a.bias)[col];
  if (a.act == ACT_RELU) s = s < 0.0f ? 0.0f : s;  // a NaN stays
  if (a.act == ACT_SILU) s = s / (1.0f + expf(-s));
  return s;
}

// Four neighbours of a row of C, from column n on.
__device__ __forceinline__ void store4(const GemmMxArgs& a, size_t row, int n, f32x4 s) {
  if (n >= a.n) return;
  const size_t at = row * a.n + n;
  if (n + 4 <= a.n) {
#pragma unroll
    for (int r = 0; r < 4; ++r) s[r] = finish(a, n + r, s[r]);
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
      const float v = finish(a, n + r, s[r]);
      if (a.c_half)
        ((uint16_t*)a.c)[at + r] = narrow<uint16_t>(v);
      else
        ((float*)a.c)[at + r] = v;
    }
}

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
template <int J>
__device__ __forceinline__ bf16x2 pair_bf16(uint32_t w, float s) {
  return __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, J);
}
__device__ __forceinline__ f16x8 eight_f16(uint32_t w, float s) {
  const h16x2 a = pair_f16<0>(w, s), b = pair_f16<1>(w, s), c = pair_f16<2>(w, s), d = pair_f16<3>(w, s);
  return f16x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}
__device__ __forceinline__ bf16x8 eight_bf16(uint32_t w, float s) {
  const bf16x2 a = pair_bf16<0>(w, s), b = pair_bf16<1>(w, s), c = pair_bf16<2>(w, s), d = pair_bf16<3>(w, s);
  return bf16x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}
// f16 elements as bf16 ones whose sum they are: the upper eight bits of the
// significand, and what is left (nothing, for an infinity).  Both are bf16
// values, the upper halves of their f32 forms.
__device__ __forceinline__ void halves(f16x8 x, bf16x8* hi, bf16x8* lo) {
  const uint4 words = __builtin_bit_cast(uint4, x);
  uint32_t h[4], l[4];
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const uint16_t b = (uint16_t)(word(words, e / 2) >> (16 * (e & 1)));
    const bool odd = (b & 0x7C00u) == 0x7C00u;  // infinities and NaN
    const float top = h2f_ieee(odd ? b : (uint16_t)(b & 0xFFF8u));
    const uint32_t t = __builtin_bit_cast(uint32_t, top);
    const uint32_t r = odd ? 0u : __builtin_bit_cast(uint32_t, h2f_ieee(b) - top);
    h[e / 2] = e % 2 ? h[e / 2] | (t & 0xFFFF0000u) : t >> 16;
    l[e / 2] = e % 2 ? l[e / 2] | (r & 0xFFFF0000u) : r >> 16;
  }
  *hi = __builtin_bit_cast(bf16x8, make_uint4(h[0], h[1], h[2], h[3]));
  *lo = __builtin_bit_cast(bf16x8, make_uint4(l[0], l[1], l[2], l[3]));
}
__device__ __forceinline__ f32x4 times_exact(uint32_t w, float s, f16x8 x, f32x4 acc) {
  bf16x8 hi, lo;
  halves(x, &hi, &lo);
  const bf16x8 v = eight_bf16(w, s);
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
// rows of A again from L2, which NT divides.
template <bool MX, int MT, int NT, bool EXACT>
__device__ __forceinline__ bool rows_sum(const GemmMxArgs& a, int n0, int from, int to, f32x4 (&acc)[NT][MT]) {
  const int lane = threadIdx.x & 63, col = lane & 15, quad = lane >> 4;
  const int blocks = (a.k + 31) / 32;
  const uint8_t *w[NT], *ws[NT], *x[MT], *xs[MT];
  bool there[MT];
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    const size_t n = min(n0 + t * 16 + col, a.n - 1);  // rows behind the end are not stored
    w[t] = a.w + n * blocks * 16;
    ws[t] = a.ws + n * blocks;
#pragma unroll
    for (int u = 0; u < MT; ++u) acc[t][u] = f32x4{};
  }
#pragma unroll
  for (int u = 0; u < MT; ++u) {
    there[u] = u * 16 + col < a.m;
    const size_t m = there[u] ? u * 16 + col : 0;
    x[u] = (const uint8_t*)a.a + (MX ? m * blocks * 16 : m * a.lda * 2);
    xs[u] = MX ? a.as + m * blocks : nullptr;
  }
  const uint32_t turn = 8 * quad + 9;  // a rotation by this takes byte `quad` to bits 30:23
  uint32_t odd = 0;                    // a factor that f16 does not hold
  for (int s0 = from; s0 < to; s0 += 4) {
    uint4 wv[NT][4], sw[NT], sx[MT];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      sw[t] = scales16(ws[t], s0 * 4, blocks);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int b = (s0 + i) * 4 + quad;
        wv[t][i] = b < blocks && s0 + i < to ? *(const uint4*)(w[t] + (size_t)b * 16) : make_uint4(0, 0, 0, 0);
      }
    }
    if constexpr (MX) {
#pragma unroll
      for (int u = 0; u < MT; ++u) sx[u] = scales16(xs[u], s0 * 4, blocks);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (s0 + i >= to) break;
      const int b = (s0 + i) * 4 + quad;
      uint32_t fw[NT];
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        const uint32_t v = word(sw[t], i);
        if constexpr (MX) {
          fw[t] = v >> (8 * quad);
        } else {
          fw[t] = __builtin_amdgcn_alignbit(v, v, turn);
          if constexpr (!EXACT) {
            const uint4 q = wv[t][i];
            const bool some = ((q.x | q.y | q.z | q.w) & 0x77777777u) != 0;
            const bool out = (fw[t] & 0x7F800000u) - (104u << 23) > (36u << 23);
            odd |= (uint32_t)((out && some) || (fw[t] & 0x7F800000u) == 0x7F800000u);
          }
        }
      }
#pragma unroll
      for (int u = 0; u < MT; ++u) {
        if constexpr (MX) {
          const bool in = there[u] && b < blocks;
          const uint4 v = in ? *(const uint4*)(x[u] + (size_t)b * 16) : make_uint4(0, 0, 0, 0);
          const uint32_t fx = in ? word(sx[u], i) >> (8 * quad) : 127u;
#pragma unroll
          for (int t = 0; t < NT; ++t) {
            const i32x8 p = {(int)wv[t][i].x, (int)wv[t][i].y, (int)wv[t][i].z, (int)wv[t][i].w, 0, 0, 0, 0};
            const i32x8 q = {(int)v.x, (int)v.y, (int)v.z, (int)v.w, 0, 0, 0, 0};
            acc[t][u] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(p, q, acc[t][u], 4, 4, 0, (int)fw[t], 0,
                                                                        (int)fx);
          }
        } else {
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int k = b * 32 + j * 8;
            const f16x8 v = there[u] && k < a.lda ? *(const f16x8*)(x[u] + (size_t)k * 2) : f16x8{};
#pragma unroll
            for (int t = 0; t < NT; ++t) {
              const float f = __builtin_bit_cast(float, fw[t]);
              if constexpr (EXACT)
                acc[t][u] = times_exact(word(wv[t][i], j), f, v, acc[t][u]);
              else
                acc[t][u] =
                    __builtin_amdgcn_mfma_f32_16x16x32_f16(eight_f16(word(wv[t][i], j), f), v, acc[t][u], 0, 0, 0);
            }
          }
        }
      }
    }
  }
  return odd != 0;
}

template <bool MX, int MT, int NT>
__global__ __launch_bounds__(MT* NT == 1 ? 1024 : 512) void gemm_mx_rows_kernel(GemmMxArgs a) {
  extern __shared__ __align__(16) f32x4 sums[];  // [waves][NT * MT][64]
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
  const int n0 = blockIdx.x * 16 * NT, steps = ((a.k + 31) / 32 + 3) / 4;
  f32x4 acc[NT][MT];
  // the waves' shares are whole groups of four steps
  const int groups = (steps + 3) / 4;
  const int from = groups * wave / waves * 4, to = min(steps, groups * (wave + 1) / waves * 4);
  const bool odd = rows_sum<MX, MT, NT, false>(a, n0, from, to, acc);
  if constexpr (!MX)
    if (__ballot(odd)) rows_sum<MX, MT, NT, true>(a, n0, from, to, acc);
  if (waves > 1) {
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
      if (m < a.m) store4(a, m, n0 + t * 16 + (lane >> 4) * 4, s);
    }
}

// A's rows at a stride of whole 16 bytes, zeros behind their ends.
__global__ __launch_bounds__(256) void pad_rows_kernel(const uint16_t* __restrict__ x, uint16_t* __restrict__ y, int m,
                                                       int k, int lda) {
  const int j = (blockIdx.x * 256 + threadIdx.x) * 8;
  if (j >= lda) return;
  for (int r = blockIdx.y; r < m; r += gridDim.y) {
    const uint16_t* p = x + (size_t)r * k + j;
    Loose<uint16_t, 8> v;
    if (j + 8 <= k) {
      v = load_loose<uint16_t, 8>(p);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) v.v[i] = j + i < k ? p[i] : (uint16_t)0;
    }
    *(Loose<uint16_t, 8>*)__builtin_assume_aligned(y + (size_t)r * lda + j, 16) = v;
  }
}

template <bool MX, int MT, int NT>
void launch_rows(hipStream_t st, const GemmMxArgs& a) {
  const int tiles = (a.n + 16 * NT - 1) / (16 * NT), groups = ((a.k + 31) / 32 + 15) / 16;
  int waves = 1;
  while (waves < (MT * NT == 1 ? 16 : 8) && waves * 2 * NT * MT <= 64 && waves < groups && tiles * waves < 4096) waves *= 2;
  const size_t lds = waves > 1 ? (size_t)waves * NT * MT * 1024 : 0;
  hipLaunchKernelGGL((gemm_mx_rows_kernel<MX, MT, NT>), dim3((unsigned)tiles), dim3(64u * waves), lds, st, a);
}

template <bool MX>
void rows(hipStream_t st, const GemmMxArgs& a) {
  if (a.m <= 16)
    launch_rows<MX, 1, 1>(st, a);
  else if (a.m <= 32)
    launch_rows<MX, 2, 2>(st, a);
  else
    launch_rows<MX, 4, 2>(st, a);
}

// --- the others -----------------------------------------------------------------

template <bool MX>
__global__ __launch_bounds__(256) void gemm_mx_plain_kernel(GemmMxArgs a) {
  const size_t blocks = (a.k + 31) / 32, total = (size_t)a.m * a.n;
  for (size_t i = (size_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (size_t)gridDim.x * 256) {
    const size_t row = i / a.n, col = i - row * a.n;
    const uint32_t* w = (const uint32_t*)a.w + col * blocks * 4;
    float sum = 0.0f;
    for (size_t b = 0; b < blocks; ++b) {
      const float sw = mx_scale(a.ws[col * blocks + b]);
      for (int j = 0; j < 4; ++j) {
        float v[8], u[8];
        mx_decode8(w[b * 4 + j], sw, v);
        if (MX) mx_decode8(((const uint32_t*)a.a)[(row * blocks + b) * 4 + j], mx_scale(a.as[row * blocks + b]), u);
        for (int e = 0; e < 8; ++e) {
          const size_t at = b * 32 + j * 8 + e;
          if (at < (size_t)a.k) sum = fmaf(MX ? u[e] : h2f_ieee(((const uint16_t*)a.a)[row * a.lda + at]), v[e], sum);
        }
      }
    }
    sum = finish(a, (int)col, sum);
    if (a.c_half)
      ((uint16_t*)a.c)[i] = narrow<uint16_t>(sum);
    else
      ((float*)a.c)[i] = sum;
  }
}

}  // namespace

size_t gemm_mx_space(const GemmMxArgs& a) {
  return a.as || a.k % 8 == 0 ? 0 : (size_t)a.m * ((a.k + 7) / 8 * 8) * 2;
}

void launch_gemm_mx(hipStream_t st, GemmMxArgs a, void* space) {
  a.lda = a.k;
  if (!a.as && a.k % 8) {
    a.lda = (a.k + 7) / 8 * 8;
    hipLaunchKernelGGL(pad_rows_kernel, dim3((unsigned)((a.lda + 2047) / 2048), (unsigned)std::min(a.m, 65535)),
                       dim3(256), 0, st, (const uint16_t*)a.a, (uint16_t*)space, a.m, a.k, a.lda);
    a.a = space;
  }
  if (a.m <= 64) {
    a.as ? rows<true>(st, a) : rows<false>(st, a);
  } else {
    const size_t total = (size_t)a.m * a.n;
    const dim3 grid((unsigned)std::min<size_t>((total + 255) / 256, 1u << 20));
    hipLaunchKernelGGL(a.as ? gemm_mx_plain_kernel<true> : gemm_mx_plain_kernel<false>, grid, dim3(256), 0, st, a);
  }
  DW_HIP(hipGetLastError());
}

}  // namespace dw
