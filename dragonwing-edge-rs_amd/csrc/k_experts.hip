// A mixture of experts around its products (k_gemm_experts.hip): which experts
// each token takes and with what weights, the choices sorted by expert, and
// the weighted sum of a token's experts' rows.
#include <algorithm>

#include "dw_common.h"
#include "mxfp4.h"

namespace dw {

namespace {

// --- routing --------------------------------------------------------------------

// Over each row of 16 lanes, the result in all of them (rotations by 8, 4, 2
// and 1 lanes).
template <int BY>
__device__ __forceinline__ uint32_t rotated(uint32_t v) {
  return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x120 + BY, 0xF, 0xF, true);
}
template <int BY>
__device__ __forceinline__ float rotated(float v) {
  return __builtin_bit_cast(float, rotated<BY>(__builtin_bit_cast(uint32_t, v)));
}
template <int BY>
__device__ __forceinline__ double rotated(double v) {
  const unsigned long long b = __builtin_bit_cast(unsigned long long, v);
  const unsigned long long lo = rotated<BY>((uint32_t)b), hi = rotated<BY>((uint32_t)(b >> 32));
  return __builtin_bit_cast(double, lo | hi << 32);
}
__device__ __forceinline__ float larger(float a, float b) { return fmaxf(a, b); }
__device__ __forceinline__ double larger(double a, double b) { return fmax(a, b); }
template <typename C>
__device__ __forceinline__ C max16(C v) {
  v = larger(v, rotated<8>(v));
  v = larger(v, rotated<4>(v));
  v = larger(v, rotated<2>(v));
  return larger(v, rotated<1>(v));
}
template <typename C>
__device__ __forceinline__ C sum16(C v) {
  v += rotated<8>(v);
  v += rotated<4>(v);
  v += rotated<2>(v);
  return v + rotated<1>(v);
}
__device__ __forceinline__ uint32_t min16(uint32_t v) {
  v = min(v, rotated<8>(v));
  v = min(v, rotated<4>(v));
  v = min(v, rotated<2>(v));
  return min(v, rotated<1>(v));
}

__device__ __forceinline__ float exponential(float x) { return expf(x); }
__device__ __forceinline__ double exponential(double x) { return exp(x); }

// exp(x - m), x <= m: 1 where both are infinite.
template <typename C>
__device__ __forceinline__ C below(C x, C m) {
  return x == m ? (C)1 : exponential(x - m);
}

// A wave's accesses of its own LDS before here go before those behind.
__device__ __forceinline__ void own_lds() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

constexpr int kMostTop = 32;

// Sixteen lanes a token, expert v * 16 + lane being value v of a lane.  C: the
// type of the choice values: f32 where they are the logits themselves, else
// f64, because scores plus biases may lie closer than f32 can tell.
template <typename C, int V, bool GROUPS>
__global__ __launch_bounds__(256) void route_kernel(RouteArgs a) {
  extern __shared__ __align__(16) double route_lds[];
  const float kNone = -INFINITY;
  const int lane = threadIdx.x & 15;
  const size_t t = (size_t)blockIdx.x * (blockDim.x / 16) + threadIdx.x / 16;
  const bool real = t < a.tokens;
  const size_t row = (real ? t : a.tokens - 1) * a.stride;
  float x[V];
  float top = kNone;
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const int e = v * 16 + lane;
    x[v] = kNone;
    if (e < a.experts) {
      const float l = a.half ? h2f_ieee(((const uint16_t*)a.x)[row + e]) : ((const float*)a.x)[row + e];
      x[v] = l > kNone ? l : kNone;  // a NaN is never chosen
    }
    top = fmaxf(top, x[v]);
  }
  top = max16(top);
  C c[V];
  constexpr bool kScores = sizeof(C) == 8;  // else choices are logits
  if constexpr (kScores) {
    C all = 1;
    if (!a.sigmoid) {
      all = 0;
#pragma unroll
      for (int v = 0; v < V; ++v) all += x[v] > kNone ? below((C)x[v], (C)top) : (C)0;
      all = sum16(all);
    }
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const int e = v * 16 + lane;
      const C p = a.sigmoid ? 1 / (1 + exponential(-(C)x[v])) : below((C)x[v], (C)top) / all;
      const C y = a.bias && e < a.experts ? p + (C)a.bias[e] : p;
      c[v] = x[v] > kNone && y > (C)kNone ? y : (C)kNone;
    }
  } else {
#pragma unroll
    for (int v = 0; v < V; ++v) c[v] = x[v];
  }
  if constexpr (GROUPS) {
    // the groups' values from LDS, 16 at a time
    const int size = a.experts / a.groups;
    C* mine = (C*)route_lds + (size_t)(threadIdx.x / 16) * (a.experts + a.groups);
    C* value = mine + a.experts;
#pragma unroll
    for (int v = 0; v < V; ++v)
      if (v * 16 + lane < a.experts) mine[v * 16 + lane] = c[v];
    own_lds();
    for (int g = lane; g < a.groups; g += 16) {
      C one = (C)kNone, two = (C)kNone;
      for (int i = 0, j = lane % size; i < size; ++i, j = j + 1 == size ? 0 : j + 1) {
        const C y = mine[g * size + j];
        two = larger(two, y < one ? y : one);
        one = larger(one, y);
      }
      value[g] = a.group_best == 2 && two > (C)kNone ? one + two : one;
    }
    own_lds();
    for (int g = lane; g < a.groups; g += 16) {
      const C y = value[g];
      int before = 0;
      for (int h = 0; h < a.groups; ++h) before += value[h] > y || (value[h] == y && h < g);
      if (before >= a.top_groups)
        for (int i = 0; i < size; ++i) mine[g * size + i] = (C)kNone;
    }
    own_lds();
#pragma unroll
    for (int v = 0; v < V; ++v)
      if (v * 16 + lane < a.experts) c[v] = mine[v * 16 + lane];
  }
  // choice j and its logit in lane j % 16
  int id[kMostTop / 16];
  float logit[kMostTop / 16];
  float best_logit = kNone;
#pragma unroll
  for (int i = 0; i < kMostTop / 16; ++i) id[i] = -1, logit[i] = kNone;
  for (int j = 0; j < a.top_k; ++j) {
    C best = c[0];
    int at = 0;
#pragma unroll
    for (int v = 1; v < V; ++v)
      if (c[v] > best) best = c[v], at = v;
    const C first = max16(best);
    const uint32_t e = min16(best == first && first > (C)kNone ? (uint32_t)(at * 16 + lane) : ~0u);
    if (__ballot(e != ~0u) == 0) break;  // the same for the wave
    float l = kNone;
#pragma unroll
    for (int v = 0; v < V; ++v)
      if (e == (uint32_t)(v * 16 + lane)) l = x[v], c[v] = (C)kNone;
    l = max16(l);
    best_logit = fmaxf(best_logit, l);
    if (e != ~0u && lane == (j & 15)) {
      if (j < 16) id[0] = (int)e, logit[0] = l;
      else id[1] = (int)e, logit[1] = l;
    }
  }
  // the weights: renormalised ones relative to the largest chosen logit, so that
  // they are sums of no vanishing terms
  float w[kMostTop / 16], sum = 0.0f, all = 1.0f;
  if (!a.sigmoid && !a.renorm) {
    all = 0.0f;
#pragma unroll
    for (int v = 0; v < V; ++v) all += x[v] > kNone ? below(x[v], top) : 0.0f;
    all = sum16(all);
  }
  const float m = a.sigmoid ? fminf(best_logit, 0.0f) : a.renorm ? best_logit : top;
#pragma unroll
  for (int i = 0; i < kMostTop / 16; ++i) {
    w[i] = 0.0f;
    if (id[i] >= 0) {
      if (!a.sigmoid)
        w[i] = below(logit[i], m);
      else if (a.renorm)
        w[i] = 1.0f / (expf(m) + expf(m - logit[i]));
      else
        w[i] = 1.0f / (1.0f + expf(-logit[i]));
    }
    sum += w[i];
  }
  if (a.renorm) all = sum16(sum);
  if (!real) return;
#pragma unroll
  for (int i = 0; i < kMostTop / 16; ++i) {
    const int j = i * 16 + lane;
    if (j >= a.top_k) continue;
    a.ids[t * a.top_k + j] = id[i];
    a.weights[t * a.top_k + j] = id[i] >= 0 ? a.scale * (w[i] / all) : 0.0f;
  }
}

template <typename C, int V>
void launch_route_v(hipStream_t st, const RouteArgs& a) {
  const int threads = a.experts <= 256 ? 256 : 64, rows = threads / 16;
  const dim3 grid((unsigned)((a.tokens + rows - 1) / rows));
  if (a.groups > 1 && a.top_groups < a.groups)
    hipLaunchKernelGGL((route_kernel<C, V, true>), grid, dim3(threads), (size_t)rows * (a.experts + a.groups) * sizeof(C), st,
                       a);
  else
    hipLaunchKernelGGL((route_kernel<C, V, false>), grid, dim3(threads), 0, st, a);
}

template <typename C>
void launch_route_c(hipStream_t st, const RouteArgs& a) {
  if (a.experts <= 16)
    launch_route_v<C, 1>(st, a);
  else if (a.experts <= 32)
    launch_route_v<C, 2>(st, a);
  else if (a.experts <= 64)
    launch_route_v<C, 4>(st, a);
  else if (a.experts <= 128)
    launch_route_v<C, 8>(st, a);
  else if (a.experts <= 256)
    launch_route_v<C, 16>(st, a);
  else if (a.experts <= 512)
    launch_route_v<C, 32>(st, a);
  else
    launch_route_v<C, 64>(st, a);
}

// --- the choices by expert ------------------------------------------------------

// A stable sort by counting.  A workgroup places a piece of the slots: where they
// go follows from how many slots before them, and in all, have each expert.
constexpr int kOrderThreads = 1024, kMostExperts = 1024;

// Lanes of the wave that hold the same id as this one (`bits` bits of it).
__device__ __forceinline__ unsigned long long same_id(int id, int bits) {
  unsigned long long same = ~0ull;
  for (int b = 0; b < bits; ++b) {
    const unsigned long long on = __ballot(id >> b & 1);
    same &= id >> b & 1 ? on : ~on;
  }
  return same;
}

// The ids [from, to) counted into count[experts] (LDS).
__device__ __forceinline__ void count_ids(const OrderArgs& a, int from, int to, int* count) {
  for (int i = from + (int)threadIdx.x; i < to; i += kOrderThreads) {
    const int id = a.ids[i];
    if ((uint32_t)id < (uint32_t)a.experts) atomicAdd(&count[id], 1);
  }
}

__global__ __launch_bounds__(kOrderThreads) void count_kernel(OrderArgs a, int piece, int* counts) {
  __shared__ int count[kMostExperts];
  for (int e = threadIdx.x; e < a.experts; e += kOrderThreads) count[e] = 0;
  __syncthreads();
  const int from = blockIdx.x * piece;
  count_ids(a, from, min(from + piece, a.slots), count);
  __syncthreads();
  for (int e = threadIdx.x; e < a.experts; e += kOrderThreads) counts[(size_t)blockIdx.x * a.experts + e] = count[e];
}

// counts: those of each piece, or null where the workgroup counts them itself.
__global__ __launch_bounds__(kOrderThreads) void order_kernel(OrderArgs a, int piece, const int* counts, int bits) {
  constexpr int kWaves = kOrderThreads / 64;
  __shared__ int all[kMostExperts], at[kMostExperts], sums[kWaves];
  __shared__ uint16_t wave_count[kWaves][kMostExperts];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int from = blockIdx.x * piece, to = min(from + piece, a.slots), pieces = gridDim.x;
  all[tid] = at[tid] = 0;
  for (int e = lane; e < kMostExperts; e += 64) wave_count[wave][e] = 0;
  __syncthreads();
  if (counts) {
    if (tid < a.experts) {
      int before = 0, sum = 0;
#pragma unroll 8
      for (int p = 0; p < pieces; ++p) {
        const int n = counts[(size_t)p * a.experts + tid];
        if (p < (int)blockIdx.x) before += n;
        sum += n;
      }
      all[tid] = sum, at[tid] = before;
    }
  } else {
    count_ids(a, 0, from, at);
    count_ids(a, 0, a.slots, all);
  }
  // this wave's slots, in order
  const int each = piece / kWaves, w0 = min(from + wave * each, to), w1 = min(w0 + each, to);
  for (int i = w0 + lane; i < w1; i += 64) {
    const int id = a.ids[i];
    if ((uint32_t)id < (uint32_t)a.experts) {
      // two counts share a word
      atomicAdd((uint32_t*)wave_count[wave] + id / 2, 1u << (16 * (id & 1)));
    }
  }
  __syncthreads();
  // where each expert's begin, and where this workgroup's do
  const int mine = all[tid];
  const int upto = sums_upto(mine);
  if (lane == 63) sums[wave] = upto;
  __syncthreads();
  int begin = upto - mine, total = 0;
  for (int w = 0; w < kWaves; ++w) {
    if (w < wave) begin += sums[w];
    total += sums[w];
  }
  if (blockIdx.x == 0 && tid < a.experts) {
    a.offsets[tid] = begin;
    if (tid == a.experts - 1) a.offsets[a.experts] = total;
  }
  int place = begin + at[tid];
  __syncthreads();
  for (int w = 0; w < kWaves; ++w) {  // of each wave: its first place
    const int n = wave_count[w][tid];
    // places are kept from the workgroup's first on, below 2^16
    wave_count[w][tid] = (uint16_t)(place - begin - at[tid]);
    place += n;
  }
  all[tid] = begin + at[tid];
  __syncthreads();
  for (int i0 = w0; i0 < w1; i0 += 64) {
    const int i = i0 + lane;
    const int id = i < w1 ? a.ids[i] : -1;
    const bool valid = (uint32_t)id < (uint32_t)a.experts;
    const unsigned long long same = same_id(valid ? id : 0, bits) & __ballot(valid);
    const int rank = __popcll(same & ((1ull << lane) - 1));
    int first = 0;
    if (valid) first = wave_count[wave][id];
    own_lds();
    if (valid && rank == 0) wave_count[wave][id] = (uint16_t)(first + __popcll(same));
    own_lds();
    if (valid) {
      const int to_place = all[id] + first + rank;
      if (to_place < a.slots) a.order[to_place] = i;
    }
  }
  // places behind the last
  for (int i = from + tid; i < to; i += kOrderThreads)
    if (i >= total) a.order[i] = -1;
}

// 4,096 slots a piece, more where that would make more than 256 of them, up to
// 65,536 (of 2^24 slots).
int piece_of(const OrderArgs& a) {
  int piece = 4096;
  while (piece < 65536 && a.slots > piece * 256) piece *= 2;
  return piece;
}
int pieces_of(const OrderArgs& a) { return (a.slots + piece_of(a) - 1) / piece_of(a); }
constexpr int kCountedApart = 4;  // pieces from which on a launch of its own counts

// --- the weighted sum -----------------------------------------------------------

// N elements (16 bytes) a thread, the token's rows one after the other.
template <typename T, int N>
__global__ __launch_bounds__(256) void combine_kernel(CombineArgs a) {
  const int i = (blockIdx.y * blockDim.x + threadIdx.x) * N;
  if (i >= a.n) return;
  const bool whole = i + N <= a.n;
  auto load = [&](const T* p) {
    Loose<T, N> v = {};
    if (whole)
      v = load_loose<T, N>(p);
    else
      for (int e = 0; i + e < a.n; ++e) v.v[e] = p[e];
    return v;
  };
  for (size_t t = (size_t)blockIdx.x * blockDim.y + threadIdx.y; t < a.tokens; t += (size_t)gridDim.x * blockDim.y) {
    float y[N] = {};
    if (a.base) {
      const Loose<T, N> v = load((const T*)a.base + t * a.n + i);
#pragma unroll
      for (int e = 0; e < N; ++e) y[e] = widen(v.v[e]);
    }
    for (int j = 0; j < a.top_k; ++j) {
      const size_t slot = t * a.top_k + j;
      if ((uint32_t)a.ids[slot] >= (uint32_t)a.experts) continue;
      const float w = a.weights[slot];
      const Loose<T, N> v = load((const T*)a.x + slot * a.n + i);
#pragma unroll
      for (int e = 0; e < N; ++e) y[e] = fmaf(w, widen(v.v[e]), y[e]);
    }
    Loose<T, N> out;
#pragma unroll
    for (int e = 0; e < N; ++e) out.v[e] = narrow<T>(y[e]);
    T* p = (T*)a.y + t * a.n + i;
    if (whole)
      store_loose<T, N>(p, out);
    else
      for (int e = 0; i + e < a.n; ++e) p[e] = out.v[e];
  }
}

template <typename T, int N>
void launch_combine_t(hipStream_t st, const CombineArgs& a) {
  const int units = (a.n + N - 1) / N;
  unsigned tx = 32;
  while (tx < 256 && tx < (unsigned)units) tx *= 2;
  const dim3 block(tx, 256 / tx);
  const dim3 grid((unsigned)std::min<size_t>((a.tokens + block.y - 1) / block.y, 1 << 20), (units + tx - 1) / tx);
  hipLaunchKernelGGL((combine_kernel<T, N>), grid, block, 0, st, a);
}

}  // namespace

void launch_route(hipStream_t st, const RouteArgs& a) {
  const bool kept = a.top_groups < a.groups;
  if (a.bias || (kept && a.group_best == 2))
    launch_route_c<double>(st, a);
  else
    launch_route_c<float>(st, a);
  DW_HIP(hipGetLastError());
}

size_t order_space(const OrderArgs& a) {
  const int pieces = pieces_of(a);
  return pieces < kCountedApart ? 0 : (size_t)pieces * a.experts * 4;
}

void launch_order(hipStream_t st, const OrderArgs& a, void* space) {
  const int pieces = pieces_of(a);
  int bits = 0;
  while (1 << bits < a.experts) ++bits;
  int* counts = pieces < kCountedApart ? nullptr : (int*)space;
  if (counts) hipLaunchKernelGGL(count_kernel, dim3(pieces), dim3(kOrderThreads), 0, st, a, piece_of(a), counts);
  hipLaunchKernelGGL(order_kernel, dim3(pieces), dim3(kOrderThreads), 0, st, a, piece_of(a), counts, bits);
  DW_HIP(hipGetLastError());
}

void launch_combine(hipStream_t st, int dtype, const CombineArgs& a) {
  if (dtype == F16)
    launch_combine_t<uint16_t, 8>(st, a);
  else
    launch_combine_t<float, 4>(st, a);
  DW_HIP(hipGetLastError());
}

}  // namespace dw
