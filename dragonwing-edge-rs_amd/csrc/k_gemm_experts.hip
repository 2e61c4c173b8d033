// Products of rows and the MXFP4 weights of their own expert: the rows' slots
// are sorted by expert, and expert e's are the places offsets[e] to
// offsets[e + 1].  The products themselves are those of one weight matrix
// (gemm_mx.h); what is here is which rows and weights a workgroup takes.  Only
// the device knows how many rows an expert has, so the grid has room for every
// case and a workgroup finds its share from the offsets.
#include <algorithm>

#include "dw_hip.h"
#include "gemm_mx_ring.h"
#include "kv_lists.h"

namespace dw {

namespace {

// A workgroup's share: some rows of an expert.
struct Share {
  int expert, first, count;  // its first place and how many it has
};

// Expert number `mine` of those that have 1 to `most` rows.  All lanes of a wave
// ask for the same.
__device__ __forceinline__ bool expert_of(const GemmExpertsArgs& x, int most, int mine, Share* s) {
  const int lane = threadIdx.x & 63;
  for (int e0 = 0; e0 < x.experts; e0 += 64) {
    const int e = e0 + lane;
    NewTokens t{0, 0};
    if (e < x.experts) t = new_tokens(x.offsets[e], x.offsets[e + 1], x.g.m);
    const unsigned long long some = __ballot(t.count > 0 && t.count <= most);
    const int n = __popcll(some);
    if (mine >= n) {
      mine -= n;
      continue;
    }
    const bool hit = (some >> lane & 1) && __popcll(some & ((1ull << lane) - 1)) == mine;
    const int src = __ffsll(__ballot(hit)) - 1;
    s->expert = e0 + src;
    s->first = __builtin_amdgcn_readlane(t.first, src);
    s->count = __builtin_amdgcn_readlane(t.count, src);
    return true;
  }
  return false;
}

// The product's arguments for one expert: its weights, scales (rows of `pitch`
// bytes) and bias.
__device__ __forceinline__ GemmMxArgs of_expert(const GemmExpertsArgs& x, int expert, int pitch) {
  GemmMxArgs a = x.g;
  const size_t rows = (size_t)expert * a.n, blocks = (a.k + 31) / 32;
  a.w += rows * blocks * 16;
  a.ws += rows * pitch;
  if (a.bias) a.bias = (const uint8_t*)a.bias + rows * (a.c_half ? 2 : 4);
  return a;
}

__device__ __forceinline__ RowList list_of(const GemmExpertsArgs& x) {
  return {x.gather ? x.order : nullptr, (uint32_t)x.g.m, (uint32_t)x.gather};
}

// C's row of a place, below 0 for none.
__device__ __forceinline__ int row_of(const GemmExpertsArgs& x, int place) {
  return x.scatter ? row_named(x.order[place], x.g.m) : place;
}

// --- experts of few rows ------------------------------------------------------------

constexpr int kFew = 16;  // the columns of a matrix instruction

// Up to 16 rows of an expert times NT x 16 of its columns (rows of W), a share of
// K, by one wave.
//
// Bound by the weights' bytes, read once, straight into the lanes that multiply
// them: a lane's operand is a block of 32 elements, four lanes side by side read
// 64 bytes of a row.  What carries it is bytes in flight: the loads of a batch (256
// elements of K) are issued before the products of the batch ahead of it, and the
// weights' first ones before the rows' list is known.  NT divides what is read of
// A again.  Times in us for 16 tokens of 8 of 64 experts x 2,816 x 2,048, 48 of them
// hit: f16 rows 39.6, MXFP4 rows 34.4 (30.1 at a copy's rate); 64 tokens of 8 of 128 x
// 4,096 x 4,096, 118 hit: 229 and 199 (215).
template <bool MX, int NT>
struct Stream {
  static constexpr int kSteps = 2;  // of 128 elements, a batch
  struct Batch {
    uint4 w[NT][kSteps];
    uint32_t sw[NT][kSteps];
    uint4 x[kSteps][MX ? 1 : 4];
    uint32_t sx[kSteps];
  };
  const GemmMxArgs& g;
  const uint8_t *w, *ws, *x, *xs;    // w, ws: the first row's, the same for all lanes
  uint32_t at_w[NT], at_s[NT];  // this lane's rows behind it
  int lane, col, quad, blocks, to;

  __device__ __forceinline__ Stream(const GemmMxArgs& args, int n0, int end) : g(args), to(end) {
    lane = threadIdx.x & 63, col = lane & 15, quad = lane >> 4, blocks = (g.k + 31) / 32;
    w = g.w + (size_t)n0 * blocks * 16;
    ws = g.ws + (size_t)n0 * blocks;
#pragma unroll
    for (int t = 0; t < NT; ++t) {  // rows behind the end are not stored
      at_s[t] = min(t * 16 + col, g.n - 1 - n0) * blocks;
      at_w[t] = (at_s[t] + quad) * 16;
    }
  }
  __device__ __forceinline__ void rows(const RowList& list, int first) {
    const size_t m = list.row(first + min(col, g.m - 1));
    x = (const uint8_t*)g.a + (MX ? (m * blocks + quad) * 16 : (m * g.lda + quad * 32) * 2);
    xs = MX ? g.as + m * blocks : nullptr;
  }
  // Steps from which on a batch needs care.
  __device__ __forceinline__ int whole() const { return min(to, MX ? blocks / 4 : g.lda / 128); }
  // The scale bytes of step s of a row: those behind its end are 127, the factor one.
  __device__ __forceinline__ uint32_t scale4(const uint8_t* row, int s) const {
    uint32_t v = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) v |= (s * 4 + j < blocks ? (uint32_t)row[s * 4 + j] : 127u) << (8 * j);
    return v;
  }
  template <bool ALL>
  __device__ __forceinline__ void load_w(Batch& b, int s) const {
#pragma unroll
    for (int t = 0; t < NT; ++t) {
#pragma unroll
      for (int i = 0; i < kSteps; ++i)
        b.w[t][i] = ALL || (s + i < to && (s + i) * 4 + quad < blocks)
                        ? *(const uint4*)(w + (size_t)(uint32_t)s * 64 + at_w[t] + i * 64)
                        : make_uint4(0, 0, 0, 0);
      if constexpr (ALL) {
        __builtin_memcpy(b.sw[t], ws + (size_t)(uint32_t)s * 4 + at_s[t], 4 * kSteps);
      } else {
#pragma unroll
        for (int i = 0; i < kSteps; ++i) b.sw[t][i] = scale4(ws + at_s[t], s + i);
      }
    }
  }
  template <bool ALL>
  __device__ __forceinline__ void load_x(Batch& b, int s) const {
    if constexpr (MX) {
#pragma unroll
      for (int i = 0; i < kSteps; ++i)
        b.x[i][0] = ALL || (s + i < to && (s + i) * 4 + quad < blocks) ? *(const uint4*)(x + (size_t)(uint32_t)s * 64 + i * 64)
                                                                     : make_uint4(0, 0, 0, 0);
      if constexpr (ALL) {
        __builtin_memcpy(b.sx, xs + (size_t)(uint32_t)s * 4, 4 * kSteps);
      } else {
#pragma unroll
        for (int i = 0; i < kSteps; ++i) b.sx[i] = scale4(xs, s + i);
      }
    } else {
#pragma unroll
      for (int i = 0; i < kSteps; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j)
          b.x[i][j] = ALL || (s + i < to && ((s + i) * 4 + quad) * 32 + j * 8 < g.lda)
                          ? *(const uint4*)(x + (size_t)(uint32_t)s * 256 + i * 256 + j * 16)
                          : make_uint4(0, 0, 0, 0);
    }
  }
  template <bool EXACT>
  __device__ __forceinline__ void multiply(const Batch& b, uint32_t* odd, f32x4 (&acc)[NT]) const {
#pragma unroll
    for (int i = 0; i < kSteps; ++i)
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        const uint4 q = b.w[t][i];
        if constexpr (MX) {
          const i32x8 p = {(int)q.x, (int)q.y, (int)q.z, (int)q.w, 0, 0, 0, 0};
          const uint4 y = b.x[i][0];
          const i32x8 v = {(int)y.x, (int)y.y, (int)y.z, (int)y.w, 0, 0, 0, 0};
          acc[t] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(p, v, acc[t], 4, 4, 0, (int)(b.sw[t][i] >> (8 * quad)), 0,
                                                                   (int)(b.sx[i] >> (8 * quad)));
        } else {
          const uint32_t fb = __builtin_amdgcn_alignbit(b.sw[t][i], b.sw[t][i], 8 * quad + 9);  // byte `quad` to bits 30:23
          const float f = __builtin_bit_cast(float, fb);
          if constexpr (!EXACT) {
            const uint32_t some = (q.x | q.y | q.z | q.w) & 0x77777777u;
            *odd |= (fb & 0x7F800000u) - (104u << 23) > (36u << 23) ? some : 0u;
          }
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const f16x8 v = __builtin_bit_cast(f16x8, b.x[i][j]);
            if constexpr (EXACT)
              acc[t] = times_exact(quarters_bf16(word(q, j), f), v, acc[t]);
            else
              acc[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(eight_f16(word(q, j), f), v, acc[t], 0, 0, 0);
          }
        }
      }
  }
  // Steps from `s` on; those of the first batch have their weights in `one`, if
  // they are whole.
  __device__ __forceinline__ uint32_t sum(int s, Batch& one, f32x4 (&acc)[NT]) const {
    uint32_t odd = 0;
    const int end = whole();
    if (s + kSteps <= end) {
      Batch two;
      load_x<true>(one, s);
      // two batches a turn, each loaded ahead of the other's products
      while (s + 3 * kSteps <= end) {
        load_w<true>(two, s + kSteps), load_x<true>(two, s + kSteps);
        __builtin_amdgcn_sched_barrier(0);
        multiply<false>(one, &odd, acc);
        __builtin_amdgcn_sched_barrier(0);
        load_w<true>(one, s + 2 * kSteps), load_x<true>(one, s + 2 * kSteps);
        __builtin_amdgcn_sched_barrier(0);
        multiply<false>(two, &odd, acc);
        __builtin_amdgcn_sched_barrier(0);
        s += 2 * kSteps;
      }
      if (s + 2 * kSteps <= end) {
        load_w<true>(two, s + kSteps), load_x<true>(two, s + kSteps);
        __builtin_amdgcn_sched_barrier(0);
        multiply<false>(one, &odd, acc);
        multiply<false>(two, &odd, acc);
        s += 2 * kSteps;
      } else {
        multiply<false>(one, &odd, acc);
        s += kSteps;
      }
    }
#pragma unroll 1
    for (; s < to; s += kSteps) {
      load_w<false>(one, s), load_x<false>(one, s);
      multiply<false>(one, &odd, acc);
    }
    return odd;
  }
  // The same in a form that holds for every factor of the weights.
  __device__ __forceinline__ void sum_exact(int s, f32x4 (&acc)[NT]) const {
    Batch b;
#pragma unroll
    for (int t = 0; t < NT; ++t) acc[t] = f32x4{};
#pragma unroll 1
    for (; s < to; s += kSteps) {
      load_w<false>(b, s), load_x<false>(b, s);
      multiply<true>(b, nullptr, acc);
    }
  }
};

// The waves of a workgroup share K, and their sums meet in LDS in order.  Of the 230 and
// 200 us of 118 experts (above), two waves make 236 and 212, eight 295 and 239.
constexpr int kRowWaves = 4;
// LOOP: workgroups take one piece of work after the other.
template <bool MX, int NT, bool LOOP>
__global__ __launch_bounds__(64 * kRowWaves) void expert_rows_kernel(GemmExpertsArgs x) {
  __shared__ __align__(16) f32x4 sums[kRowWaves][NT][64];
  using S = Stream<MX, NT>;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int tiles = (x.g.n + 16 * NT - 1) / (16 * NT), steps = ((x.g.k + 31) / 32 + 3) / 4;
  const int batches = (steps + S::kSteps - 1) / S::kSteps;
  const int from = batches * wave / kRowWaves * S::kSteps, to = min(steps, batches * (wave + 1) / kRowWaves * S::kSteps);
  for (unsigned id = blockIdx.x;; id += gridDim.x) {
    const int item = id / tiles, n0 = (id - item * tiles) * 16 * NT;
    Share s;
    if (!expert_of(x, kFew, item, &s)) return;
    GemmMxArgs a = of_expert(x, s.expert, (x.g.k + 31) / 32);
    a.m = s.count;
    S stream(a, n0, to);
    typename S::Batch first;
    if (from + S::kSteps <= stream.whole()) stream.template load_w<true>(first, from);
    stream.rows(list_of(x), s.first);
    f32x4 acc[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) acc[t] = f32x4{};
    const uint32_t odd = stream.sum(from, first, acc);
    if constexpr (!MX)
      if (__ballot(odd != 0)) stream.sum_exact(from, acc);
#pragma unroll
    for (int t = 0; t < NT; ++t) sums[wave][t][lane] = acc[t];
    __syncthreads();
    const int m = lane & 15, row = m < s.count ? row_of(x, s.first + m) : -1;
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      if (row < 0 || t % kRowWaves != wave) continue;
      f32x4 c = sums[0][t][lane];
#pragma unroll
      for (int i = 1; i < kRowWaves; ++i) c += sums[i][t][lane];
      const int n = n0 + t * 16 + (lane >> 4) * 4;
      store4<true>(a, row, n, c, bias4(a, n));
    }
    if (!LOOP) return;
    __syncthreads();
  }
}

// --- experts of more rows -----------------------------------------------------------

// Tile `id` of the grid: which expert's, and which rows and columns of it.
template <class T>
__device__ __forceinline__ bool tile_of(const GemmExpertsArgs& x, int id, int tiles_n, Share* s, int* m0, int* n0) {
  const int lane = threadIdx.x & 63;
  NewTokens t{0, 0};
  auto tiles = [&](int e) {
    t = NewTokens{0, 0};
    if (e < x.experts) t = new_tokens(x.offsets[e], x.offsets[e + 1], x.g.m);
    return t.count > x.few ? (t.count + T::kRowsA - 1) / T::kRowsA : 0;
  };
  int all = 0;
  for (int e0 = 0; e0 < x.experts; e0 += 64) all += __builtin_amdgcn_readlane(sums_upto(tiles(e0 + lane)), 63);
  int tile;
  if (!tile_number(id, all, tiles_n, &tile)) return false;
  const int row = tile / tiles_n;
  int before = 0;
  for (int e0 = 0; e0 < x.experts; e0 += 64) {
    const int n = tiles(e0 + lane), upto = sums_upto(n);
    const unsigned long long hit = __ballot(row >= before + upto - n && row < before + upto);
    if (hit) {
      const int src = __ffsll(hit) - 1;
      s->expert = e0 + src;
      s->first = __builtin_amdgcn_readlane(t.first, src);
      s->count = __builtin_amdgcn_readlane(t.count, src);
      const int rows = __builtin_amdgcn_readlane(n, src);
      const int at = tile - (before + __builtin_amdgcn_readlane(upto - n, src)) * tiles_n;
      // eight rows of tiles wide, so that operands are shared in the XCD's L2
      constexpr int kBand = 8;
      const int band = at / (kBand * tiles_n), high = min(kBand, rows - band * kBand);
      const int off = at - band * kBand * tiles_n;
      *m0 = (band * kBand + off % high) * T::kRowsA;
      *n0 = off / high * T::kRowsW;
      return true;
    }
    before += __builtin_amdgcn_readlane(upto, 63);
  }
  return false;
}

// The sums of rows from r0 of a part of a tile in LDS to C: four columns a lane, a
// step's rows apart, kAtOnce rows whose reads and activations overlap.
template <class OUT, int ACT, int kLine, int kStep, int kPart, int kTall, int kFull>
__device__ __forceinline__ void store_part(const GemmMxArgs& a, const uint8_t* lds, const int* rows, int piece, int n,
                                           f32x4 bias) {
  constexpr int kAtOnce = 4, N = ACT == ACT_SWIGLU ? 2 : 4;
  static_assert(kPart % (kAtOnce * kStep) == 0, "whole steps");
  const int line = ACT == ACT_SWIGLU ? a.n / 2 : a.n, c0 = ACT == ACT_SWIGLU ? n / 2 : n;  // n and a.n are even there
  auto silu_of = [](float s) { return std::is_same<OUT, float>::value ? silu(s) : silu_f16(s); };
#pragma unroll 1
  for (int r0 = threadIdx.x / (kLine / 16); r0 < kPart; r0 += kAtOnce * kStep) {
    int row[kAtOnce];
    f32x4 v[kAtOnce];
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i) {
      const int r = r0 + i * kStep;
      row[i] = rows[r / kTall * kFull + r % kTall];
      v[i] = *(const f32x4*)(lds + r * kLine + (piece ^ (r & 7)) * 16) + bias;
    }
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i) {
      Loose<OUT, N> y;
#pragma unroll
      for (int j = 0; j < N; ++j) {
        const float s = ACT == ACT_SWIGLU ? silu_of(v[i][2 * j % 4]) * v[i][(2 * j + 1) % 4]
                        : ACT == ACT_SILU ? silu_of(v[i][j])
                        : ACT == ACT_RELU && v[i][j] < 0.0f ? 0.0f : v[i][j];  // a NaN stays
        y.v[j] = narrow<OUT>(s);
      }
      OUT* to = (OUT*)a.c + (size_t)(uint32_t)row[i] * (uint32_t)line + c0;
      if (row[i] < 0) continue;
      if (c0 + N <= line)
        store_loose<OUT, N>(to, y);
      else
#pragma unroll
        for (int j = 0; j < N - 1; ++j)
          if (c0 + j < line) to[j] = y.v[j];
    }
  }
}

// A tile's sums to C, through LDS (behind `rows`, which keeps C's rows), in kPieces
// parts: a wave's stores cover rows of C whole, and the code of an activation is
// short (written out for every sum, a 256 x 256 tile of f16 rows with SiLU spent 17 of 134 us
// on it at K = 4,096, and spends 9).  A row's pieces of 16 bytes stand at their index
// xor the row's, so that eight rows' writes meet all banks.
template <int WM, int WN, int TM, int TN, int kPieces>
__device__ __forceinline__ void store_tile(const GemmMxArgs& a, uint8_t* lds, const int* rows, int n0,
                                           const f32x4 (&acc)[TN][TM]) {
  constexpr int kLine = WN * TN * 64, kLanes = kLine / 16, kTall = TM / kPieces * 16, kStep = WM * WN * 64 / kLanes;
  static_assert(TM % kPieces == 0, "whole parts");
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, wm = wave % WM, wn = wave / WM;
  const int col = lane & 15, quad = lane >> 4;
  const int piece = threadIdx.x % kLanes, n = n0 + piece * 4;
  const f32x4 bias = bias4(a, n);
#pragma unroll 1
  for (int part = 0; part < kPieces; ++part) {
    if (part) __syncthreads();
#pragma unroll
    for (int p = 0; p < kPieces; ++p) {
      if (p != part) continue;
#pragma unroll
      for (int u = 0; u < TM / kPieces; ++u)
#pragma unroll
        for (int t = 0; t < TN; ++t) {
          const int r = wm * kTall + u * 16 + col;
          *(f32x4*)(lds + r * kLine + (((wn * TN + t) * 4 + quad) ^ (r & 7)) * 16) = acc[t][p * (TM / kPieces) + u];
        }
    }
    __syncthreads();
    auto store = [&](auto out, auto act) {
      store_part<decltype(out), act.value, kLine, kStep, WM * kTall, kTall, TM * 16>(a, lds, rows + part * kTall, piece,
                                                                                     n, bias);
    };
    auto as = [&](auto act) { a.c_half ? store(uint16_t(), act) : store(float(), act); };
    if (a.act == ACT_SWIGLU)
      as(std::integral_constant<int, ACT_SWIGLU>());
    else if (a.act == ACT_SILU)
      as(std::integral_constant<int, ACT_SILU>());
    else if (a.act == ACT_RELU)
      as(std::integral_constant<int, ACT_RELU>());
    else
      as(std::integral_constant<int, ACT_NONE>());
  }
}

// C's rows of a tile's, below 0 for none, to LDS.
template <int ROWS>
__device__ __forceinline__ void rows_of(const GemmExpertsArgs& x, int m0, int end, int* rows) {
  if (threadIdx.x < ROWS) rows[threadIdx.x] = m0 + (int)threadIdx.x < end ? row_of(x, m0 + threadIdx.x) : -1;
}

template <bool MX, int WM, int WN, int TM, int TN>
__global__ __launch_bounds__(WM* WN * 64) void expert_tile_kernel(GemmExpertsArgs x, int tiles_n) {
  using T = Tile<MX, WM, WN, TM, TN, true>;
  extern __shared__ __align__(16) uint8_t lds[];
  Share s;
  int m0, n0;
  if (!tile_of<T>(x, blockIdx.x, tiles_n, &s, &m0, &n0)) return;
  GemmMxArgs a = of_expert(x, s.expert, (x.g.k + 31) / 32);
  m0 += s.first;
  a.m = s.first + s.count;
  const int stages = (a.k + T::kDepth - 1) / T::kDepth;
  int* rows = (int*)(lds + T::kLds);
  rows_of<T::kRowsA>(x, m0, a.m, rows);
  f32x4 acc[TN][TM];
  const T t(a, lds, m0, n0, list_of(x));
  const uint32_t far = t.template sum<false>(0, stages, acc);
  if constexpr (!MX) {
    if (__syncthreads_or(far != 0) && __syncthreads_or(t.outside(0, stages))) t.template sum<true>(0, stages, acc);
  }
  constexpr int kBytes = T::kRowsA * T::kRowsW * 4, kPieces = kBytes <= T::kLds ? 1 : 2;
  static_assert(kBytes <= kPieces * T::kLds && T::kRowsA <= WM * WN * 64, "fits");
  store_tile<WM, WN, TM, TN, kPieces>(a, lds, rows, n0, acc);
}

template <bool MX>
__global__ __launch_bounds__(512) void expert_ring_kernel(GemmExpertsArgs x, int tiles_n) {
  using R = Ring<MX>;
  extern __shared__ __align__(16) uint8_t lds[];
  Share s;
  int m0, n0;
  if (!tile_of<R>(x, blockIdx.x, tiles_n, &s, &m0, &n0)) return;
  GemmMxArgs a = of_expert(x, s.expert, x.g.pitch);
  m0 += s.first;
  a.m = s.first + s.count;
  int* rows = (int*)(lds + R::kLds);
  rows_of<R::kRowsA>(x, m0, a.m, rows);
  f32x4 acc[R::TN][R::TM];
  const R r(a, lds, m0, n0, list_of(x));
  const uint32_t far = r.template sum<false>(acc);
  if constexpr (!MX) {
    if (__syncthreads_or(far != 0) && __syncthreads_or(r.outside())) r.template sum<true>(acc);
  }
  static_assert(R::kRowsA * R::kRowsW * 4 <= 2 * R::kLds, "fits");
  store_tile<2, 4, R::TM, R::TN, 2>(a, lds, rows, n0, acc);
}

// How a product is cut, and where its workspace lies.  Which experts have how many
// rows only the device knows: expert_rows_kernel takes those of up to kFew, and the
// tiles of the others have a height that suits the mean.  In us: 32 rows on average, f16 rows
// 111 in tiles of 64 x 128 and 157 in 128 x 128, MXFP4 rows 79 in 64 x 64 and 90 in 128 x 128;
// 128 rows 237 and 145 in 128 x 128, 262 and 177 in 256 x 256; 175 rows 466 and 228 in 128
// x 128, 487 and 228 in 256 x 256; 1,024 rows 1,047 and 537 in 128 x 128, 813 and 389
// in 256 x 256 with their scales laid out anew.
struct Plan {
  int height, width;  // of the tiles of experts of more than kFew rows; 0: there are none
  size_t tiles;       // of them at most
  bool pads;          // rows of scales laid out anew, of whole 16 bytes
  size_t a_rows, rows_at, scales_a, scales_w, bytes;
};
constexpr int kRare = 64;  // rows an expert has on average, from which on those of kFew are rare

// Columns / 16 of a workgroup of expert_rows_kernel: four where that leaves workgroups
// enough (64 tokens of 8 of 118 experts x 4,096 x 4,096: f16 rows 230 us, with two 270, MXFP4
// rows 200 and 213), two for fewer (a token of 8 experts x 2,816 x 2,048: 8.9 and 7.9 us,
// with four 9.8 and 9.0).
int tiles_a_row(const GemmMxArgs& g) { return (g.as ? (size_t)g.m * g.n >= (size_t)1 << 21 : g.m >= 64) ? 4 : 2; }

Plan plan(const GemmExpertsArgs& x) {
  Plan p{};
  const GemmMxArgs& g = x.g;
  auto take = [&](size_t bytes) {
    const size_t at = p.bytes;
    p.bytes += (bytes + 255) / 256 * 256;
    return at;
  };
  p.a_rows = x.gather ? g.m / x.gather : g.m;
  if (g.m > kFew) {
    const int mean = g.m / x.experts;
    p.height = mean >= 192 ? 256 : mean >= kRare ? 128 : 64;
    p.width = p.height == 64 && !g.as ? 128 : p.height;
    // whole tiles, and one that is not for each expert that has some
    const size_t most = g.m / p.height + std::min(x.experts, g.m / (kFew + 1));
    p.tiles = most * ((g.n + p.width - 1) / p.width);
    if (p.tiles >= (size_t)1 << 23)  // of up to 512 threads: a grid has under 2^32
      fail(DW_ERR_UNSUPPORTED, "gemm_mxfp4_experts: more than 2^23 tiles");
  }
  const size_t rows_n = 16 * tiles_a_row(g);
  if ((g.n + rows_n - 1) / rows_n * std::min(x.experts, g.m) >= (size_t)1 << 24)  // of 256 threads
    fail(DW_ERR_UNSUPPORTED, "gemm_mxfp4_experts: a grid of more than 2^32 threads");
  const size_t blocks = (g.k + 31) / 32, pitch = (blocks + 15) / 16 * 16;
  if (!g.as && g.k % 8) p.rows_at = take(p.a_rows * ((g.k + 7) / 8 * 8) * 2);
  p.pads = p.height == 256 && blocks % 16;
  if (p.pads) {
    if (g.as) p.scales_a = take(p.a_rows * pitch);
    p.scales_w = take((size_t)x.experts * g.n * pitch);
  }
  return p;
}

// Where experts of few rows are rare, 512 workgroups look for them, all that run at a
// time: the 8,192 of 65,536 x 4,096 x 4,096 for 128 experts take 9 us to find none.  Where
// they are most of the work, a workgroup for each piece is faster (64 x 8 of 118 experts,
// MXFP4 rows x 4,096 x 4,096: 199 us, 212 in a loop).
template <bool MX, int NT>
void launch_expert_rows(hipStream_t st, const GemmExpertsArgs& x) {
  const unsigned all = (unsigned)((x.g.n + 16 * NT - 1) / (16 * NT) * std::min(x.experts, x.g.m));
  constexpr bool kLoops = MX || NT == 4;  // kRare f16 rows come with NT = 4
  if (kLoops && x.g.m / x.experts >= kRare)
    hipLaunchKernelGGL((expert_rows_kernel<MX, NT, kLoops>), dim3(std::min(all, 512u)), dim3(64 * kRowWaves), 0, st, x);
  else
    hipLaunchKernelGGL((expert_rows_kernel<MX, NT, false>), dim3(all), dim3(64 * kRowWaves), 0, st, x);
}

template <bool MX>
void launch_expert_rows(hipStream_t st, const GemmExpertsArgs& x) {
  tiles_a_row(x.g) == 4 ? launch_expert_rows<MX, 4>(st, x) : launch_expert_rows<MX, 2>(st, x);
}

template <bool MX, int WM, int WN, int TM, int TN>
void launch_expert_tiles(hipStream_t st, const GemmExpertsArgs& x, size_t tiles) {
  using T = Tile<MX, WM, WN, TM, TN, true>;
  auto* k = expert_tile_kernel<MX, WM, WN, TM, TN>;
  hipLaunchKernelGGL(k, dim3((unsigned)tiles), dim3(WM * WN * 64), T::kLds + T::kRowsA * 4, st, x,
                     (x.g.n + T::kRowsW - 1) / T::kRowsW);
}

template <bool MX>
void launch_expert_rings(hipStream_t st, const GemmExpertsArgs& x, size_t tiles) {
  hipLaunchKernelGGL(expert_ring_kernel<MX>, dim3((unsigned)tiles), dim3(512), Ring<MX>::kLds + 1024, st, x,
                     (x.g.n + 255) / 256);
}

}  // namespace

size_t gemm_experts_space(const GemmExpertsArgs& x) { return plan(x).bytes; }

void launch_gemm_experts(hipStream_t st, GemmExpertsArgs x, void* space) {
  const Plan p = plan(x);
  GemmMxArgs& g = x.g;
  char* base = (char*)space;
  const int blocks = (g.k + 31) / 32, words = (blocks + 15) / 16 * 4;
  g.lda = (g.k + 7) / 8 * 8;
  g.pitch = words * 4;
  auto groups = [](size_t units) { return (unsigned)std::min<size_t>((units + 255) / 256, 4096); };
  Pads pads{};
  pads.m = (int)p.a_rows, pads.k = g.k, pads.lda = g.lda, pads.blocks = blocks, pads.words = words;
  if (!g.as && g.k % 8) {
    pads.x = (const uint16_t*)g.a;
    g.a = pads.x_to = (uint16_t*)(base + p.rows_at);
    pads.first = groups(p.a_rows * (g.lda / 8));
  }
  const GemmExpertsArgs few = x;  // scales as they are
  unsigned others = 0;
  if (p.pads) {
    if (g.as) {
      pads.s[0] = g.as, pads.rows[0] = p.a_rows;
      g.as = (const uint8_t*)(pads.s_to[0] = (uint32_t*)(base + p.scales_a));
      pads.first = groups(p.a_rows * words);
    }
    pads.s[1] = g.ws, pads.rows[1] = (size_t)x.experts * g.n;
    g.ws = (const uint8_t*)(pads.s_to[1] = (uint32_t*)(base + p.scales_w));
    others = groups(pads.rows[1] * words);
  }
  launch_pads(st, pads, others);
  g.as ? launch_expert_rows<true>(st, few) : launch_expert_rows<false>(st, few);
  x.few = kFew;
  if (p.height == 256)
    g.as ? launch_expert_rings<true>(st, x, p.tiles) : launch_expert_rings<false>(st, x, p.tiles);
  else if (p.height == 128)
    g.as ? launch_expert_tiles<true, 2, 2, 4, 4>(st, x, p.tiles) : launch_expert_tiles<false, 2, 2, 4, 4>(st, x, p.tiles);
  else if (p.height)
    g.as ? launch_expert_tiles<true, 1, 4, 4, 1>(st, x, p.tiles) : launch_expert_tiles<false, 2, 2, 2, 4>(st, x, p.tiles);
  DW_HIP(hipGetLastError());
}

}  // namespace dw
