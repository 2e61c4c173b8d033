// Products of rows and the MXFP4 weights of their own expert: the rows' slots
// are sorted by expert, and expert e's are the places offsets[e] to
// offsets[e + 1].  The products themselves are those of one weight matrix
// (gemm_mx.h); what is here is which rows and weights a workgroup takes.  Only
// the device knows how many rows an expert has, so the grid has room for every
// case and a workgroup finds its share from the offsets.
#include <algorithm>

#include "dw_hip.h"
#include "gemm_mx.h"
#include "kv_lists.h"

namespace dw {

namespace {

// A workgroup's share: some rows of an expert.
struct Share {
  int expert, first, count;  // its first place and how many it has
};

// Expert number `mine` of those that have 1 to `most` rows.  All lanes of a wave
// ask for the same.
__device__ __forceinline__ bool few_rows_expert(const GemmExpertsArgs& x, int most, int mine, Share* s) {
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
  if (!x.scatter) return place;
  const int r = x.order[place];
  return r < x.g.m ? r : -1;
}

// --- experts of few rows ------------------------------------------------------------

constexpr int kFew = 16;

template <bool MX, bool FEW>
__device__ __forceinline__ void rows_of_expert(const GemmExpertsArgs& x, const GemmMxArgs& a, const Share& s, f32x4* sums) {
  using R = Rows<MX, 1, 1, FEW, true>;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
  const int n0 = blockIdx.x * 16, steps = ((a.k + 31) / 32 + 3) / 4, groups = (steps + 3) / 4;
  const int from = groups * wave / waves * 4, to = min(steps, groups * (wave + 1) / waves * 4);
  f32x4 acc[1][1];
  const R r(a, n0, (uint8_t*)sums + wave * 4 * R::kFewLine, list_of(x), s.first);
  const uint32_t odd = r.template sum<false>(from, to, acc);
  if constexpr (!MX)
    if (__ballot(odd != 0)) r.template sum<true>(from, to, acc);
  f32x4 c = acc[0][0];
  if (waves > 1) {
    if (FEW) __syncthreads();  // the rows' place becomes the sums'
    sums[wave * 64 + lane] = c;
    __syncthreads();
    if (wave) return;
    for (int i = 1; i < waves; ++i) c += sums[i * 64 + lane];
  }
  const int m = lane & 15, n = n0 + (lane >> 4) * 4;
  if (m >= s.count) return;
  const int row = row_of(x, s.first + m);
  if (row >= 0) store4<true>(a, row, n, c, bias4(a, n));
}

template <bool MX>
__global__ __launch_bounds__(512) void expert_rows_kernel(GemmExpertsArgs x) {
  extern __shared__ __align__(16) f32x4 sums[];
  Share s;
  if (!few_rows_expert(x, kFew, blockIdx.y, &s)) return;
  GemmMxArgs a = of_expert(x, s.expert, (x.g.k + 31) / 32);
  a.m = s.count;
  if (!MX && s.count <= 4)
    rows_of_expert<MX, true>(x, a, s, sums);
  else
    rows_of_expert<MX, false>(x, a, s, sums);
}

// --- experts of many rows -----------------------------------------------------------

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
  // Neighbouring workgroups go to the 8 XCDs in turn: each takes a run of tiles.
  const int total = all * tiles_n, per = total / 8, rest = total % 8, xcd = id % 8, in = id / 8;
  if (in >= per + (xcd < rest)) return false;
  const int tile = xcd * per + min(xcd, rest) + in, row = tile / tiles_n;
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

template <bool MX, int WM, int WN, int TM, int TN>
__global__ __launch_bounds__(WM* WN * 64) void expert_tile_kernel(GemmExpertsArgs x, int tiles_n) {
  using T = Tile<MX, WM, WN, TM, TN, true>;
  extern __shared__ __align__(16) uint8_t lds[];
  Share s;
  int m0, n0;
  if (!tile_of<T>(x, blockIdx.x, tiles_n, &s, &m0, &n0)) return;
  GemmMxArgs a = of_expert(x, s.expert, x.g.pitch);
  m0 += s.first;
  a.m = s.first + s.count;
  const int stages = (a.k + T::kDepth - 1) / T::kDepth;
  f32x4 acc[TN][TM];
  const T t(a, lds, m0, n0, list_of(x));
  const uint32_t far = t.template sum<false>(0, stages, acc);
  if constexpr (!MX) {
    if (__syncthreads_or(far != 0) && __syncthreads_or(t.outside(0, stages))) t.template sum<true>(0, stages, acc);
  }
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int m1 = m0 + wave % WM * TM * 16 + (lane & 15), n1 = n0 + wave / WM * TN * 16 + (lane >> 4) * 4;
  f32x4 bias[TN];
#pragma unroll
  for (int i = 0; i < TN; ++i) bias[i] = bias4(a, n1 + i * 16);
#pragma unroll
  for (int u = 0; u < TM; ++u) {
    if (m1 + u * 16 >= a.m) continue;
    const int row = row_of(x, m1 + u * 16);
    if (row < 0) continue;
#pragma unroll
    for (int i = 0; i < TN; ++i) store4<true>(a, row, n1 + i * 16, acc[i][u], bias[i]);
  }
}

// How a product is cut, and where its workspace lies.
struct Plan {
  bool rows;   // experts of up to kFew rows apart
  int height;  // of the others' tiles, square ones; 0: there are none
  size_t tiles;  // of them at most
  size_t a_rows, rows_at, scales_a, scales_w, bytes;
};
Plan plan(const GemmExpertsArgs& x) {
  Plan p{};
  const GemmMxArgs& g = x.g;
  auto take = [&](size_t bytes) {
    const size_t at = p.bytes;
    p.bytes += (bytes + 255) / 256 * 256;
    return at;
  };
  p.a_rows = x.gather ? g.m / x.gather : g.m;
  p.rows = g.m <= kFew || g.m / x.experts <= 2 * kFew;
  p.height = g.m <= kFew ? 0 : g.m / x.experts >= 256 ? 256 : 128;
  if (p.height) {
    // whole tiles, and one that is not for each expert that has some
    const size_t most = g.m / p.height + std::min(x.experts, p.rows ? g.m / (kFew + 1) : g.m);
    p.tiles = most * ((g.n + p.height - 1) / p.height);
    if (p.tiles >= (size_t)1 << 23)  // of up to 512 threads: a grid has under 2^32
      fail(DW_ERR_UNSUPPORTED, "gemm_mxfp4_experts: more than 2^23 tiles");
  }
  const size_t blocks = (g.k + 31) / 32, pitch = (blocks + 15) / 16 * 16;
  if (!g.as && g.k % 8) p.rows_at = take(p.a_rows * ((g.k + 7) / 8 * 8) * 2);
  if (p.height && blocks % 16) {
    if (g.as) p.scales_a = take(p.a_rows * pitch);
    p.scales_w = take((size_t)x.experts * g.n * pitch);
  }
  return p;
}

template <bool MX>
void launch_expert_rows(hipStream_t st, const GemmExpertsArgs& x) {
  const int tiles = (x.g.n + 15) / 16, groups = ((x.g.k + 31) / 32 + 15) / 16, items = std::min(x.experts, x.g.m);
  int waves = 1;
  while (waves < 8 && waves < groups && (long long)tiles * items * waves < 4096) waves *= 2;
  const size_t lds = (size_t)waves * (MX ? 1024 : 4 * Rows<MX, 1, 1, true, true>::kFewLine);
  hipLaunchKernelGGL(expert_rows_kernel<MX>, dim3((unsigned)tiles, (unsigned)items), dim3(64u * waves), lds, st, x);
}

template <bool MX, int WM, int WN, int TM, int TN>
void launch_expert_tiles(hipStream_t st, const GemmExpertsArgs& x, size_t tiles) {
  using T = Tile<MX, WM, WN, TM, TN, true>;
  auto* k = expert_tile_kernel<MX, WM, WN, TM, TN>;
  hipLaunchKernelGGL(k, dim3((unsigned)tiles), dim3(WM * WN * 64), T::kLds, st, x, (x.g.n + T::kRowsW - 1) / T::kRowsW);
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
  GemmExpertsArgs few = x;
  if (!g.as && g.k % 8) {
    pads.x = (const uint16_t*)g.a;
    g.a = few.g.a = pads.x_to = (uint16_t*)(base + p.rows_at);
    pads.first = groups(p.a_rows * (g.lda / 8));
  }
  unsigned others = 0;
  if (p.height && blocks % 16) {
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
  if (p.rows) g.as ? launch_expert_rows<true>(st, few) : launch_expert_rows<false>(st, few);
  x.few = p.rows ? kFew : 0;
  if (p.height == 256)
    g.as ? launch_expert_tiles<true, 2, 4, 8, 4>(st, x, p.tiles) : launch_expert_tiles<false, 2, 4, 8, 4>(st, x, p.tiles);
  else if (p.height)
    g.as ? launch_expert_tiles<true, 2, 2, 4, 4>(st, x, p.tiles) : launch_expert_tiles<false, 2, 2, 4, 4>(st, x, p.tiles);
  DW_HIP(hipGetLastError());
}

}  // namespace dw
