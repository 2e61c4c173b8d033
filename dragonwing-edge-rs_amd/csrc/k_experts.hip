// A mixture of experts around its products (k_gemm_experts.hip): which experts
// each token takes and with what weights, the choices sorted by expert, and
// the weighted sum of a token's experts' rows.
#include <algorithm>
#include <type_traits>
#include <utility>

#include "dw_common.h"
#include "mxfp4.h"

namespace dw {

namespace {

// --- routing --------------------------------------------------------------------

// A lane's number moved by data-parallel primitives (within each row of 16 lanes).
template <int CTRL>
__device__ __forceinline__ uint32_t moved(uint32_t v) {
  return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xF, 0xF, true);
}
template <int CTRL>
__device__ __forceinline__ float moved(float v) {
  return __builtin_bit_cast(float, moved<CTRL>(__builtin_bit_cast(uint32_t, v)));
}
__device__ __forceinline__ float larger(float a, float b) { return fmaxf(a, b); }
__device__ __forceinline__ uint32_t larger(uint32_t a, uint32_t b) { return max(a, b); }
// Over the L lanes of a token, the same result in all of them: exchanges with the
// lane beside, two on, and mirrored in 8 and 16 lanes.
template <int L, typename T, typename F>
__device__ __forceinline__ T over(T v, F f) {
  if constexpr (L >= 2) v = f(v, moved<0xB1>(v));
  if constexpr (L >= 4) v = f(v, moved<0x4E>(v));
  if constexpr (L >= 8) v = f(v, moved<0x141>(v));
  if constexpr (L >= 16) v = f(v, moved<0x140>(v));
  if constexpr (L == 64) {
    v = f(v, __shfl_xor(v, 16));
    v = f(v, __shfl_xor(v, 32));
  }
  return v;
}
template <int L, typename T>
__device__ __forceinline__ T largest(T v) {
  return over<L>(v, [](T a, T b) { return larger(a, b); });
}
template <int L, typename T>
__device__ __forceinline__ T total(T v) {
  return over<L>(v, [](T a, T b) { return a + b; });
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
constexpr float kNone = -INFINITY;  // of experts that are not chosen

// Whole numbers in the order of f32 numbers, and back.  Those of numbers above -inf
// are above kLowest.
constexpr uint32_t kLowest = 0x007FFFFFu;
__device__ __forceinline__ uint32_t ordered(float f) {
  const uint32_t b = __builtin_bit_cast(uint32_t, f);
  return b ^ ((uint32_t)((int)b >> 31) | 0x80000000u);
}
__device__ __forceinline__ float unordered(uint32_t k) {
  return __builtin_bit_cast(float, k & 0x80000000u ? k ^ 0x80000000u : ~k);
}

// Batcher's odd-even merges: the pairs that sort V numbers, in order.
template <int V>
struct Pairs {
  int n = 0;
  int first[V * 8] = {}, second[V * 8] = {};
  constexpr Pairs() {
    for (int p = 1; p < V; p *= 2)
      for (int q = p; q >= 1; q /= 2)
        for (int j = q % p; j + q < V; j += 2 * q)
          for (int i = 0; i < q && i + j + q < V; ++i)
            if ((i + j) / (2 * p) == (i + j + q) / (2 * p)) first[n] = i + j, second[n++] = i + j + q;
  }
};
// The keys of a lane, largest first.  (The pairs are expanded by the compiler's front
// end: a register's number must be a constant.)
template <int V, size_t... S>
__device__ __forceinline__ void sort_down(uint32_t (&k)[V], std::index_sequence<S...>) {
  constexpr Pairs<V> kPairs;
  auto order = [&](uint32_t& a, uint32_t& b) {
    const uint32_t c = max(a, b);
    b = min(a, b), a = c;
  };
  (order(k[kPairs.first[S]], k[kPairs.second[S]]), ...);
}
template <int V>
__device__ __forceinline__ void sort_down(uint32_t (&k)[V]) {
  if constexpr (V > 1) sort_down(k, std::make_index_sequence<(size_t)Pairs<V>().n>());
}

// LDS of a wave in 8 bytes: f64 values of a token's experts and groups, its choices
// and 64 experts to choose from, or f32 values of all its tokens.
template <int L>
__host__ __device__ __forceinline__ size_t route_space(const RouteArgs& a) {
  const size_t n = a.experts + a.groups, one = n + (kMostTop + 64) / 2, all = n * (64 / L) / 2;
  return one > all ? one : all;
}

// L lanes have a token's row, values lane * V to lane * V + V - 1 each.
template <int L, int V>
struct Router {
  const RouteArgs& a;
  int lane;    // of the token's
  float x[V];  // logits; kNone for NaN and behind the end, no -0
  float top;   // the largest, of a softmax

  __device__ __forceinline__ Router(const RouteArgs& args, size_t row) : a(args), lane(threadIdx.x & (L - 1)) {
    if (a.half)
      load((const uint16_t*)a.x + row, x);
    else
      load((const float*)a.x + row, x);
    top = kNone;
#pragma unroll
    for (int v = 0; v < V; ++v) x[v] = fmaxf(x[v] + 0.0f, kNone);  // a NaN is never chosen, and -0 is the same as 0
    if (!a.sigmoid) {
#pragma unroll
      for (int v = 0; v < V; ++v) top = fmaxf(top, x[v]);
      top = largest<L>(top);
    }
  }
  template <typename T>
  __device__ __forceinline__ void load(const T* row, float (&to)[V]) const {
    const int e = lane * V;
    if (e + V <= a.experts) {
      const Loose<T, V> l = load_loose<T, V>(row + e);
#pragma unroll
      for (int v = 0; v < V; ++v) to[v] = widen(l.v[v]);
    } else {
#pragma unroll
      for (int v = 0; v < V; ++v) to[v] = e + v < a.experts ? widen(row[e + v]) : kNone;
    }
  }

  // Values by which experts are chosen, scores and biases, and what a score may be off:
  // in roundings (2^-24) of the largest score, a sigmoid by 4 (exponent, its product,
  // sum, reciprocal), one of a softmax by those and the sum's V + 5.  (The errors of the
  // sum's terms, 12 at most for 1,024 experts, are common to all scores, as are the sum's and
  // the reciprocal's: of two scores they count once, and twice this is more than all.)
  __device__ __forceinline__ float values(const float (&bias)[V], float (&c)[V]) const {
    constexpr float kLog2e = 1.44269504f;
    float all = 1.0f;
    if (!a.sigmoid) {
      all = 0.0f;
#pragma unroll
      for (int v = 0; v < V; ++v) {
        c[v] = x[v] == top ? 1.0f : __builtin_amdgcn_exp2f((x[v] - top) * kLog2e);
        all += x[v] > kNone ? c[v] : 0.0f;
      }
      all = __builtin_amdgcn_rcpf(total<L>(all));
#pragma unroll
      for (int v = 0; v < V; ++v) c[v] *= all;
    } else {
#pragma unroll
      for (int v = 0; v < V; ++v) c[v] = __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(x[v] * -kLog2e));
    }
#pragma unroll
    for (int v = 0; v < V; ++v) c[v] = x[v] > kNone ? fmaxf(c[v] + bias[v], kNone) : kNone;
    return (a.sigmoid ? 5.0f : V + 10.0f) * 0x1p-24f * all;
  }
  // Whether values of this size (the larger of two magnitudes) that are `gap` apart may
  // be in the other order: scores are off by `off`, and sums round once.
  static __device__ __forceinline__ bool near(float gap, float size, float off, float keys) {
    return !(gap > 2 * off + size * (0x1p-23f + keys));
  }

  // Leaves the values of the groups that are kept; true if values off by `off` might
  // give others.  mine: LDS of this token.
  __device__ __forceinline__ bool keep_groups(float (&c)[V], float off, float* mine) const {
    const int size = a.experts / a.groups, each = size / V;
    float dropped = kNone, kept = INFINITY, most = 0.0f;  // most: the largest magnitude in a sum
    if (L >= 8 && L <= 16 && each * V == size && (each & (each - 1)) == 0) {
      // a group is 1, 2, 4 or 8 lanes
      float one = c[0], two = kNone;
#pragma unroll
      for (int v = 1; v < V; ++v) two = fmaxf(two, fminf(one, c[v])), one = fmaxf(one, c[v]);
      auto join = [&](float o, float t) { two = fmaxf(fminf(one, o), fmaxf(two, t)), one = fmaxf(one, o); };
      if (each >= 2) join(moved<0xB1>(one), moved<0xB1>(two));
      if (each >= 4) join(moved<0x4E>(one), moved<0x4E>(two));
      if (each >= 8) join(moved<0x141>(one), moved<0x141>(two));
      const bool both = a.group_best == 2 && two > kNone;
      const float y = both ? one + two : one;
      most = fmaxf(one > kNone ? fabsf(one) : 0.0f, both ? fabsf(two) : 0.0f);
      // lanes of groups that come before this one: those of the token in turn
      int before = 0;
      const int shift = __ffs(each) - 1, group = lane >> shift;
      float z = y;
#pragma unroll
      for (int i = 1; i < L; ++i) {
        z = next(z);
        before += z > y || (z == y && ((lane + i) & (L - 1)) >> shift < group);
      }
      const bool in = before < a.top_groups * each;
      kept = in ? y : INFINITY, dropped = in ? kNone : y;
#pragma unroll
      for (int v = 0; v < V; ++v) c[v] = in ? c[v] : kNone;
    } else {
      float* value = mine + a.experts;
#pragma unroll
      for (int v = 0; v < V; ++v)
        if (lane * V + v < a.experts) mine[lane * V + v] = c[v];
      own_lds();
      for (int g = lane; g < a.groups; g += L) {
        float one = kNone, two = kNone;
        for (int i = 0, j = lane % size; i < size; ++i, j = j + 1 == size ? 0 : j + 1) {
          const float y = mine[g * size + j];
          two = fmaxf(two, fminf(one, y)), one = fmaxf(one, y);
        }
        const bool both = a.group_best == 2 && two > kNone;
        value[g] = both ? one + two : one;
        most = fmaxf(most, fmaxf(one > kNone ? fabsf(one) : 0.0f, both ? fabsf(two) : 0.0f));
      }
      own_lds();
      for (int g = lane; g < a.groups; g += L) {
        const float y = value[g];
        int before = 0;
        for (int h = 0; h < a.groups; ++h) before += value[h] > y || (value[h] == y && h < g);
        if (before < a.top_groups) {
          kept = fminf(kept, y);
        } else {
          dropped = fmaxf(dropped, y);
          for (int i = 0; i < size; ++i) mine[g * size + i] = kNone;
        }
      }
      own_lds();
#pragma unroll
      for (int v = 0; v < V; ++v)
        if (lane * V + v < a.experts) c[v] = mine[lane * V + v];
      own_lds();
    }
    dropped = largest<L>(dropped), kept = -largest<L>(-kept), most = largest<L>(most);
    // two sums of two values each: a value is rounded by 2^-24 of `most`, a sum by twice that, so
    // that two sums may be 8 x 2^-24 of it off, and four times what a score may be
    return dropped > kNone && near(kept - dropped, 4 * most, 2 * off, 0.0f);
  }
  // The number of the token's next lane.
  static __device__ __forceinline__ float next(float v) {
    if constexpr (L == 16) return moved<0x12F>(v);  // a rotation to the right by 15
    // 8 lanes: a rotation of all 16, and of the others' by 8, which the last lane takes
    const float f = moved<0x12F>(v), g = moved<0x127>(v);
    return (threadIdx.x & 7) == 7 ? g : f;
  }

  // The largest by keys of 32 bits, which want values without -0: each lane sorts its own,
  // and the largest first one is taken top_k times; choice j comes to lane j % L,
  // id[j / L].  WHOLE: the values are f16 numbers and keys hold them and their expert,
  // else a value's upper bits and the place in the lane, which leaves out log2 V bits
  // of 24.  True if values, off by `off`, lie closer than keys tell apart: the chosen
  // ones are then not below `least` (in lane 0).  KEEP: how many of a lane's keys may be taken.
  static constexpr int kEach = kMostTop / L > 0 ? kMostTop / L : 1;
  template <int KEEP, bool WHOLE>
  __device__ __forceinline__ bool choose(const float (&c)[V], float off, int (&id)[kEach], float* least) const {
    constexpr uint32_t kLow = V - 1;
    uint32_t k[V];
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const uint32_t e = lane * V + v;
      // f16 numbers leave 13 bits of an f32 one
      const uint32_t key = WHOLE ? (ordered(c[v]) & ~0x1FFFu) | (0x1FFFu - e) : (ordered(c[v]) & ~kLow) | (kLow - v);
      k[v] = c[v] > kNone ? key : e;  // experts that are not chosen have keys of their own, too
    }
    sort_down(k);
    const int base = (threadIdx.x & 63) - lane;
    uint32_t taken[kEach];
    int owner[kEach];
    bool twice = false;  // some token's largest key stood in two lanes
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      taken[i] = 0, owner[i] = 0;
      if (i * L >= a.top_k) continue;
      const int most = min(L, a.top_k - i * L);
#pragma unroll 1
      for (int j = 0; j < most; ++j) {
        const uint32_t first = largest<L>(k[0]);
        const unsigned long long hits = __ballot(k[0] == first);
        const bool here = lane == j;
        if constexpr (!WHOLE) {
          twice |= __popcll(hits) != 64 / L;
          const int from = L == 64 ? __ffsll(hits) - 1 : __ffs((uint32_t)(hits >> base)) - 1;
          owner[i] = here ? from : owner[i];
        }
        taken[i] = here ? first : taken[i];
        // the owner's next key moves up (by masks: a choice between two of an array's
        // numbers would become one number that is looked up)
        const uint32_t moves = k[0] == first ? ~0u : 0u;
#pragma unroll
        for (int v = 0; v + 1 < KEEP; ++v) k[v] = (k[v + 1] & moves) | (k[v] & ~moves);
        k[KEEP - 1] &= ~moves;
      }
    }
#pragma unroll
    for (int i = 0; i < kEach; ++i)
      id[i] = taken[i] <= kLowest ? -1 : WHOLE ? (int)(0x1FFFu - (taken[i] & 0x1FFFu)) : owner[i] * V + (int)(kLow - (taken[i] & kLow));
    if constexpr (WHOLE) return false;
    {
      const int j = a.top_k - 1;
      uint32_t of = 0;
#pragma unroll
      for (int i = 0; i < kEach; ++i) of = j / L == i ? taken[i] : of;
      of = __shfl(of, base + (j & (L - 1)));
      const float v = unordered(of & ~kLow);
      *least = of > kLowest && fabsf(v) < INFINITY ? v - (2 * off + fabsf(v) * 0x1p-22f) : kNone;
    }
    // each choice and the one before it, and the last one and the next that was not taken
    const uint32_t next = largest<L>(k[0]);
    bool close = twice;
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      if (i * L >= a.top_k) continue;
      const int j = i * L + lane;
      // all lanes take part in both
      const uint32_t beside = __shfl(taken[i], base + (lane ? lane - 1 : 0)), ahead = __shfl(taken[i > 0 ? i - 1 : 0], base + L - 1);
      const uint32_t up = lane ? beside : ahead;
      auto same = [&](uint32_t high, uint32_t low) {
        const float h = unordered(high & ~kLow), l = unordered(low & ~kLow);
        return low > kLowest && (off > 0.0f ? near(h - l, fmaxf(fabsf(h), fabsf(l)), off, V * 0x1p-23f) : h == l);
      };
      close |= j > 0 && j < a.top_k && same(up, taken[i]);
      close |= j == a.top_k - 1 && same(taken[i], next);
    }
    return close;
  }
};

// A token's choices by a whole wave, from values as they are compared: scores and biases
// in 64 bits, or logits.  None is below `least`.  values: LDS for experts + groups of
// them; ids: for kMostTop choices and 64 more.
template <bool SCORES>
__device__ __forceinline__ void choose_exactly(const RouteArgs& a, size_t row, float least, double* values, int* ids) {
  const int lane = threadIdx.x & 63;
  const double none = kNone;
  auto logit = [&](int e) {
    const float l = a.half ? h2f_ieee(((const uint16_t*)a.x)[row + e]) : ((const float*)a.x)[row + e];
    return l > kNone ? l : kNone;
  };
  auto over_wave = [](double v, auto f) {
#pragma unroll
    for (int i = 1; i < 64; i *= 2) v = f(v, __shfl_xor(v, i));
    return v;
  };
  auto most = [](double p, double q) { return p > q ? p : q; };
  double top = none, all = 1;
  if (SCORES && !a.sigmoid) {
    for (int e = lane; e < a.experts; e += 64) top = most(top, logit(e));
    top = over_wave(top, most);
    all = 0;
    for (int e = lane; e < a.experts; e += 64)
      if (logit(e) > kNone) all += below((double)logit(e), top);
    all = over_wave(all, [](double p, double q) { return p + q; });
  }
  for (int e = lane; e < a.experts; e += 64) {
    const double x = logit(e);
    double y = x;
    if (SCORES) {
      y = a.sigmoid ? 1 / (1 + exp(-x)) : below(x, top) / all;
      if (a.bias) y += (double)a.bias[e];
    }
    values[e] = x > none && y > none ? y : none;
  }
  own_lds();
  if (a.top_groups < a.groups) {
    double* of = values + a.experts;
    const int size = a.experts / a.groups;
    for (int g = lane; g < a.groups; g += 64) {
      double one = none, two = none;
      for (int i = 0; i < size; ++i) {
        const double y = values[g * size + i];
        two = most(two, y < one ? y : one), one = most(one, y);
      }
      of[g] = a.group_best == 2 && two > none ? one + two : one;
    }
    own_lds();
    for (int g = lane; g < a.groups; g += 64) {
      int before = 0;
      for (int h = 0; h < a.groups; ++h) before += of[h] > of[g] || (of[h] == of[g] && h < g);
      if (before >= a.top_groups)
        for (int i = 0; i < size; ++i) values[g * size + i] = none;
    }
    own_lds();
  }
  // those that may be chosen, usually one or two more than top_k: each counts the ones
  // that come before it
  int* some = ids + kMostTop;
  double bound = least;
  int n = 0;
  for (int turn = 0; turn < 2; ++turn) {
    n = 0;
    for (int e0 = 0; e0 < a.experts; e0 += 64) {
      const int e = e0 + lane;
      const bool in = e < a.experts && values[e] > none && values[e] >= bound;
      const unsigned long long all_in = __ballot(in);
      const int at = n + __popcll(all_in & ((1ull << lane) - 1));
      if (in && at < 64) some[at] = e;
      n += __popcll(all_in);
    }
    own_lds();
    if (n <= 64 || turn == 1) break;
    // choice top_k of the lanes' largest has top_k - 1 of them before it
    double best = none;
    for (int e = lane; e < a.experts; e += 64) best = most(best, values[e]);
    int before = 0;
    for (int i = 0; i < 64; ++i) {
      const double z = __shfl(best, i);
      before += z > best || (z == best && i < lane);
    }
    bound = __shfl(best, __ffsll(__ballot(before == a.top_k - 1)) - 1);
  }
  if (n <= 64) {
    if (lane < a.top_k) ids[lane] = -1;
    own_lds();
    if (lane < n) {
      const int e = some[lane];
      const double y = values[e];
      int before = 0;
      for (int i = 0; i < n; ++i) {
        const double z = values[some[i]];
        before += z > y || (z == y && some[i] < e);
      }
      if (before < a.top_k) ids[before] = e;
    }
    own_lds();
    return;
  }
  for (int j = 0; j < a.top_k; ++j) {
    double best = none;
    int at = 0x10000;
    for (int e = lane; e < a.experts; e += 64)
      if (values[e] > best) best = values[e], at = e;
    const double first = over_wave(best, most);
    at = best == first ? at : 0x10000;
#pragma unroll
    for (int i = 1; i < 64; i *= 2) at = min(at, __shfl_xor(at, i));
    if (lane == 0) {
      ids[j] = at < 0x10000 ? at : -1;
      if (at < 0x10000) values[at] = none;
    }
    own_lds();
  }
}

// L lanes a token.  SCORES: experts, or groups of them, are chosen by scores
// and biases, else by the logits.  Scores and biases may lie closer than f32 can
// tell: rows in which they do (some in a thousand, of scores that are no ties) are
// decided again in 64 bits, rows of f32 logits by comparing these as they are.
//
// Bound by instructions: 32,768 f32 rows of 256 take 13 us by their logits (10.7 of
// f16 ones, 7 us their bytes), 23 with sigmoids and biases, and 33 to 35 in 8 groups.  A
// wave that decides one row again takes some us more than the others.
template <int L, int V, bool SCORES, bool GROUPS>
__global__ __launch_bounds__(256) void route_kernel(RouteArgs a) {
  extern __shared__ __align__(16) double route_lds[];
  const size_t t = (size_t)blockIdx.x * (blockDim.x / L) + threadIdx.x / L;
  const bool real = t < a.tokens;
  const size_t row = (real ? t : a.tokens - 1) * a.stride;
  using R = Router<L, V>;
  // of a wave: f64 values of one token and its choices, or f32 ones of each
  double* wave = route_lds + (size_t)(threadIdx.x / 64) * route_space<L>(a);
  int id[R::kEach];
  float all = 1.0f, top;
  {
    const R r(a, row);
    float c[V], off = 0.0f;
    top = r.top;
    if (!a.sigmoid && !a.renorm) {
      all = 0.0f;
#pragma unroll
      for (int v = 0; v < V; ++v) all += r.x[v] > kNone ? below(r.x[v], top) : 0.0f;
      all = total<L>(all);
    }
    if constexpr (SCORES) {
      float bias[V] = {};
      if (a.bias) r.load(a.bias, bias);
      off = r.values(bias, c);
    } else {
#pragma unroll
      for (int v = 0; v < V; ++v) c[v] = r.x[v];
    }
    bool close = false;
    float least = kNone;
    if constexpr (GROUPS) close = r.keep_groups(c, off, (float*)wave + (size_t)(threadIdx.x & 63) / L * (a.experts + a.groups)) && SCORES;
    auto choose = [&](auto whole) {
      constexpr bool kWhole = decltype(whole)::value;
      return V > 9 && a.top_k <= 8 ? r.template choose<(V > 9 ? 9 : V), kWhole>(c, off, id, &least)
                                     : r.template choose<V, kWhole>(c, off, id, &least);
    };
    if (!SCORES && a.half) {
      choose(std::true_type());
    } else {
      const bool groups = close;
      close |= choose(std::false_type());
      least = groups ? kNone : least;  // of groups that may be others
    }
    for (unsigned long long left = __ballot(close); left;) {
      const int first = (__ffsll(left) - 1) / L * L;  // lane of the next token
      int* ids = (int*)(wave + a.experts + a.groups);
      own_lds();
      choose_exactly<SCORES>(a, ((size_t)__builtin_amdgcn_readlane((int)(row >> 32), first) << 32) |
                                    (uint32_t)__builtin_amdgcn_readlane((int)row, first),
                             __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, least), first)), wave, ids);
      if ((int)(threadIdx.x & 63) / L * L == first)
#pragma unroll
        for (int i = 0; i < R::kEach; ++i)
          if (i * L + r.lane < a.top_k) id[i] = ids[i * L + r.lane];
      left &= ~((L == 64 ? ~0ull : (1ull << (L & 63)) - 1) << first);
    }
  }
  // The weights, relative to the largest chosen logit where they are renormalised, so
  // that none of the sums' terms vanish.
  const int lane = threadIdx.x & (L - 1);
  float logit[R::kEach], w[R::kEach], best = kNone, sum = 0.0f;
#pragma unroll
  for (int i = 0; i < R::kEach; ++i) {
    logit[i] = kNone;
    if (i * L < a.top_k && id[i] >= 0)
      logit[i] = a.half ? h2f_ieee(((const uint16_t*)a.x)[row + id[i]]) : ((const float*)a.x)[row + id[i]];
    best = fmaxf(best, logit[i]);
  }
  best = largest<L>(best);
  const float m = a.sigmoid ? fminf(best, 0.0f) : a.renorm ? best : top;
#pragma unroll
  for (int i = 0; i < R::kEach; ++i) {
    w[i] = 0.0f;
    if (i * L < a.top_k && id[i] >= 0) {
      if (!a.sigmoid)
        w[i] = below(logit[i], m);
      else if (a.renorm)
        w[i] = 1.0f / (expf(m) + expf(m - logit[i]));
      else
        w[i] = 1.0f / (1.0f + expf(-logit[i]));
    }
    sum += w[i];
  }
  if (a.renorm) all = total<L>(sum);
  if (!real) return;
#pragma unroll
  for (int i = 0; i < R::kEach; ++i) {
    const int j = i * L + lane;
    if (j >= a.top_k) continue;
    a.ids[t * a.top_k + j] = id[i];
    a.weights[t * a.top_k + j] = id[i] >= 0 ? a.scale * (w[i] / all) : 0.0f;
  }
}

template <int L, int V, bool SCORES>
void launch_route_v(hipStream_t st, const RouteArgs& a) {
  const int rows = 256 / L;
  const dim3 grid((unsigned)((a.tokens + rows - 1) / rows));
  auto* k = a.top_groups < a.groups ? route_kernel<L, V, SCORES, true> : route_kernel<L, V, SCORES, false>;
  hipLaunchKernelGGL(k, grid, dim3(256), 4 * 8 * route_space<L>(a), st, a);
}

// Up to 256 experts 16 a lane, so that a wave has as many tokens as it can: its
// instructions are the bound.
template <bool SCORES>
void launch_route_s(hipStream_t st, const RouteArgs& a) {
  if (a.experts <= 16)
    launch_route_v<4, 4, SCORES>(st, a);
  else if (a.experts <= 32)
    launch_route_v<4, 8, SCORES>(st, a);
  else if (a.experts <= 64)
    launch_route_v<4, 16, SCORES>(st, a);
  else if (a.experts <= 128)
    launch_route_v<8, 16, SCORES>(st, a);
  else if (a.experts <= 256)
    launch_route_v<16, 16, SCORES>(st, a);
  else if (a.experts <= 512)
    launch_route_v<64, 8, SCORES>(st, a);
  else
    launch_route_v<64, 16, SCORES>(st, a);
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

// counts: those of each piece, or null where the workgroup counts them itself.  EACH:
// a lane's slots, kept in registers; 0: any number, read twice.
template <int EACH>
__global__ __launch_bounds__(kOrderThreads) void order_kernel(OrderArgs a, int piece, const int* counts, int bits) {
  constexpr int kWaves = kOrderThreads / 64;
  __shared__ int all[kMostExperts], at[kMostExperts], sums[kWaves];
  __shared__ uint16_t wave_count[kWaves][kMostExperts];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int from = blockIdx.x * piece, to = min(from + piece, a.slots), pieces = gridDim.x;
  // this wave's slots, in order
  const int each = piece / kWaves, w0 = min(from + wave * each, to), w1 = min(w0 + each, to);
  int id[EACH ? EACH : 1], rank[EACH ? EACH : 1];
#pragma unroll
  for (int u = 0; u < EACH; ++u) {
    const int i = w0 + u * 64 + lane;
    id[u] = i < w1 ? a.ids[i] : -1;
  }
  all[tid] = at[tid] = 0;
  for (int e = lane; e < kMostExperts / 2; e += 64) ((uint32_t*)wave_count[wave])[e] = 0;
  __syncthreads();
  // The number of this wave's slots ahead of lane's that have its id, and one more in
  // the count of the id for each.
  auto count = [&](int of) {
    const bool valid = (uint32_t)of < (uint32_t)a.experts;
    const unsigned long long same = same_id(valid ? of : 0, bits) & __ballot(valid);
    const int ahead = __popcll(same & ((1ull << lane) - 1));
    int before = 0;
    if (valid) before = wave_count[wave][of];
    own_lds();
    if (valid && ahead == 0) wave_count[wave][of] = (uint16_t)(before + __popcll(same));
    own_lds();
    return valid ? before + ahead : -1;
  };
  if constexpr (EACH > 0) {
#pragma unroll
    for (int u = 0; u < EACH; ++u) rank[u] = count(id[u]);
  } else {
    for (int i = w0 + lane; i < w1; i += 64) {
      const int of = a.ids[i];
      // two counts share a word
      if ((uint32_t)of < (uint32_t)a.experts) atomicAdd((uint32_t*)wave_count[wave] + of / 2, 1u << (16 * (of & 1)));
    }
  }
  if (counts) {
    // several threads an expert, each some of the pieces
    const int several = kOrderThreads / a.experts, e = tid % a.experts, share = tid / a.experts;
    if (share < several) {
      int before = 0, sum = 0;
#pragma unroll 8
      for (int p = share; p < pieces; p += several) {
        const int n = counts[(size_t)p * a.experts + e];
        before += p < (int)blockIdx.x ? n : 0;
        sum += n;
      }
      atomicAdd(&all[e], sum), atomicAdd(&at[e], before);
    }
  } else if (pieces > 1) {
    count_ids(a, 0, from, at);
    count_ids(a, 0, a.slots, all);
  }
  __syncthreads();
  if (pieces == 1)
#pragma unroll
    for (int w = 0; w < kWaves; ++w) all[tid] += wave_count[w][tid];
  // where each expert's begin, and where this workgroup's do
  const int mine = all[tid];
  const int upto = sums_upto(mine);
  if (lane == 63) sums[wave] = upto;
  __syncthreads();
  int begin = upto - mine, total = 0;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    if (w < wave) begin += sums[w];
    total += sums[w];
  }
  if (blockIdx.x == 0 && tid < a.experts) {
    a.offsets[tid] = begin;
    if (tid == a.experts - 1) a.offsets[a.experts] = total;
  }
  int ahead = 0;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {  // of each wave: its first place, from the workgroup's on, below 2^16
    const int n = wave_count[w][tid];
    wave_count[w][tid] = (uint16_t)ahead;
    ahead += n;
  }
  all[tid] = begin + at[tid];
  __syncthreads();
  auto put = [&](int of, int place, int i) {
    if (place >= 0 && all[of] + place < a.slots) a.order[all[of] + place] = i;
  };
  if constexpr (EACH > 0) {
#pragma unroll
    for (int u = 0; u < EACH; ++u) {
      const int of = rank[u] >= 0 ? id[u] : 0;
      put(of, rank[u] >= 0 ? wave_count[wave][of] + rank[u] : -1, w0 + u * 64 + lane);
    }
  } else {
    for (int i0 = w0; i0 < w1; i0 += 64) {
      const int of = i0 + lane < w1 ? a.ids[i0 + lane] : -1, place = count(of);
      put(place >= 0 ? of : 0, place, i0 + lane);
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
// Pieces from which on a launch of its own counts; below, each workgroup counts them all
// by itself.  2,048 slots 6.5 us (8.4 with the launch), 12,288 8.2 to 9.3 (8.8), 16,384 9.0
// (10.5 without), 32,000 9.8 (14.9).
constexpr int kCountedApart = 4;

// --- the weighted sum -----------------------------------------------------------

// N neighbours of a token's row, from column i on: eight of its experts' rows in flight.
template <typename T, int N>
__device__ __forceinline__ void combine(const CombineArgs& a, size_t t, int i) {
  const int32_t* ids = a.ids + t * a.top_k;
  const float* weights = a.weights + t * a.top_k;
  const T* x = (const T*)a.x + t * a.top_k * a.n + i;
  float y[N] = {};
  if (a.base) {
    const Loose<T, N> v = load_loose<T, N>((const T*)a.base + t * a.n + i);
#pragma unroll
    for (int e = 0; e < N; ++e) y[e] = widen(v.v[e]);
  }
  int j0 = 0;
  auto some = [&](auto rows) {
    constexpr int kRows = decltype(rows)::value;
    Loose<T, N> v[kRows];
    float w[kRows];
    bool in[kRows];
#pragma unroll
    for (int j = 0; j < kRows; ++j) {
      in[j] = (uint32_t)ids[j0 + j] < (uint32_t)a.experts;
      w[j] = weights[j0 + j];
    }
    // rows of no expert are not read: another stands in, and counts nothing
#pragma unroll
    for (int j = 0; j < kRows; ++j) v[j] = load_loose<T, N>(in[j] ? x + (size_t)(j0 + j) * a.n : (const T*)a.x + i);
#pragma unroll
    for (int j = 0; j < kRows; ++j)
      if (in[j])
#pragma unroll
        for (int e = 0; e < N; ++e) y[e] = fmaf(w[j], widen(v[j].v[e]), y[e]);
    j0 += kRows;
  };
  while (a.top_k - j0 >= 8) some(std::integral_constant<int, 8>());
  if (a.top_k - j0 >= 4) some(std::integral_constant<int, 4>());
  if (a.top_k - j0 >= 2) some(std::integral_constant<int, 2>());
  if (a.top_k - j0 >= 1) some(std::integral_constant<int, 1>());
  Loose<T, N> out;
#pragma unroll
  for (int e = 0; e < N; ++e) out.v[e] = narrow<T>(y[e]);
  store_loose<T, N>((T*)a.y + t * a.n + i, out);
}

// N elements (16 bytes) a thread, the last ones of a row one by one.  Bound by the
// rows' bytes.  WAVES: a wave has one token, whose ids and weights are scalars then.
template <typename T, int N, bool WAVES>
__global__ __launch_bounds__(256) void combine_kernel(CombineArgs a) {
  const int i = (blockIdx.y * blockDim.x + threadIdx.x) * N;
  if (i >= a.n) return;
  for (size_t t0 = (size_t)blockIdx.x * blockDim.y + threadIdx.y; t0 < a.tokens; t0 += (size_t)gridDim.x * blockDim.y) {
    const size_t t = WAVES ? (size_t)__builtin_amdgcn_readfirstlane((int)t0) : t0;
    if (i + N <= a.n) {
      combine<T, N>(a, t, i);
    } else {
#pragma unroll 1
      for (int e = i; e < a.n; ++e) combine<T, 1>(a, t, e);
    }
  }
}

template <typename T, int N>
void launch_combine_t(hipStream_t st, const CombineArgs& a) {
  const int units = (a.n + N - 1) / N;
  unsigned tx = 16;
  while (tx < 256 && tx < (unsigned)units) tx *= 2;
  const dim3 block(tx, 256 / tx);
  const dim3 grid((unsigned)std::min<size_t>((a.tokens + block.y - 1) / block.y, 1 << 20), (units + tx - 1) / tx);
  auto* k = tx >= 64 ? combine_kernel<T, N, true> : combine_kernel<T, N, false>;
  hipLaunchKernelGGL(k, grid, block, 0, st, a);
}

}  // namespace

void launch_route(hipStream_t st, const RouteArgs& a) {
  if (a.bias || (a.top_groups < a.groups && a.group_best == 2))
    launch_route_s<true>(st, a);
  else
    launch_route_s<false>(st, a);
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
  auto* k = piece_of(a) == 4096 ? order_kernel<4> : order_kernel<0>;
  hipLaunchKernelGGL(k, dim3(pieces), dim3(kOrderThreads), 0, st, a, piece_of(a), counts, bits);
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
