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

#include "gemm_mx.h"

namespace dw {

namespace {

constexpr int kFewRows = 32;

// --- a few rows -----------------------------------------------------------------

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

void launch_pads(hipStream_t st, const Pads& p, unsigned others) {
  if (p.first + others) hipLaunchKernelGGL(pad_kernel, dim3(p.first + others), dim3(256), 0, st, p);
}

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
  launch_pads(st, pads, others);
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
