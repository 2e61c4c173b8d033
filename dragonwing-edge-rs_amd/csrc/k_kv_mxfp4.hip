// Attention over a cache of keys and values in MXFP4 pages, and what writes
// the cache.
//
// A page holds page_size rows of each kv head, [page][head][slot][d / 2]
// bytes and [page][head][slot][d / 32] scales: the rows are MXFP4 rows of d
// elements (mxfp4.h), so the cache's values can be read back as such rows.
#include <algorithm>

#include "dw_common.h"
#include "kv_lists.h"
#include "mxfp4.h"

namespace dw {

namespace {

// The sequence that a token belongs to: how many sequences end at or before
// it.  All threads of a workgroup ask for the same token.
__device__ __forceinline__ int sequence_of(const int32_t* start, int batch, int t, int* lds) {
  if (threadIdx.x == 0) *lds = 0;
  __syncthreads();
  int n = 0;
  for (int b = threadIdx.x; b < batch; b += blockDim.x) n += start[b + 1] <= t;
  if (n) atomicAdd(lds, n);
  __syncthreads();
  return *lds;
}

// The new token's place: its page and slot, or false where the table or the
// lengths give it none.
__device__ __forceinline__ bool place_of(const KvArgs& a, int seq, int t, size_t* row) {
  if (seq >= a.batch || t < a.start[seq]) return false;
  const long long pos = (long long)a.len[seq] - a.start[seq + 1] + t;
  if (pos < 0 || pos >= (long long)a.max_pages << a.page_shift) return false;
  const int page = a.table[(size_t)seq * a.max_pages + (pos >> a.page_shift)];
  if (page < 0 || page >= a.num_pages) return false;
  *row = ((size_t)page * a.kv_heads << a.page_shift) + (pos & ((1 << a.page_shift) - 1));
  return true;
}

// One token a workgroup, eight elements a thread's step: read 2 bytes an
// element, written 17/32.  4,269 tokens of 8 heads x 128: 9.3 us (2.4 TB/s: each
// workgroup first finds its token's sequence and page, three loads one after
// the other); 64 single tokens 5.5 us.  The scale is at least 2^-23, so that every value of
// the cache is an f16 value.
__global__ __launch_bounds__(256) void kv_append_kernel(KvArgs a, const uint16_t* __restrict__ k, size_t k_stride,
                                                        size_t k_off, const uint16_t* __restrict__ v, size_t v_stride,
                                                        size_t v_off) {
  __shared__ int found;
  const int t = blockIdx.x;
  const int seq = sequence_of(a.start, a.batch, t, &found);
  size_t row;
  if (!place_of(a, seq, t, &row)) return;
  const int each = a.d / 8, units = 2 * a.kv_heads * each;
  for (int u = threadIdx.x; u < units; u += 256) {
    const bool is_v = u >= units / 2;
    const int w = is_v ? u - units / 2 : u, h = w / each, j = w - h * each;
    const uint16_t* p = (is_v ? v + t * v_stride + v_off : k + t * k_stride + k_off) + (size_t)h * a.d + j * 8;
    const Loose<uint16_t, 8> l = load_loose<uint16_t, 8>(p);
    float x[8];
    uint32_t big = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      x[i] = widen(l.v[i]);
      big = max(big, __builtin_bit_cast(uint32_t, x[i]) & 0x7FFFFFFFu);
    }
    const uint32_t b = mx_scale_byte(max_of_quad(big), 127 - 23);
    const size_t at = row + ((size_t)h << a.page_shift);
    (is_v ? a.vc : a.kc)[at * each + j] = b == 255u ? 0u : mx_encode8(x, mx_scale(b));
    if ((j & 3) == 0) (is_v ? a.vs : a.ks)[at * (each / 4) + j / 4] = (uint8_t)b;
  }
}

// A share of the work: some steps of the keys of an item, a tile of rows (new
// tokens of one sequence x heads of one kv head).
struct Split {
  int seq, token, count;  // the tile's first token and how many it has
  int kv_head, head;      // head: the tile's first
  int index, of;          // this split of the item's
  int slot;               // the item's first place in the workspace, where it has several splits
  int item;               // and its place among such items
  int first, steps;       // steps before this split, and its own
  long long pos, len;     // position of the tile's first token, keys of the sequence
};

// Which split number `mine` is; LAST: counted from the end.  Every item of a
// sequence has the same number of steps; all steps over the splits wanted is a
// split's length, so that long and short sequences share the chip evenly
// whatever their lengths, which only the device knows.  One load a 64
// sequences.  *joined: how many items have several splits (for split 0).
//
// An item has n = ceil(steps / length) splits: all items under the number of
// items + `waves`, and the items that have two or more under 2 `waves`.
constexpr long long kNever = 1ll << 62;
template <bool LAST>
__device__ __forceinline__ bool plan(const KvArgs& a, const AttnArgs& g, const SplitArgs& p, int mine, Split* s,
                                     int* joined) {
  const int lane = threadIdx.x & 63, heads = p.head_tiles * a.kv_heads;
  const int most = a.max_pages << a.page_shift;
  int first, items, steps, count, len, raw;
  bool on = true;  // tiles of 128 rows
  auto load = [&](int b) {
    first = count = len = raw = 0;
    if (b >= a.batch) return;
    const NewTokens t = new_tokens(a.start[b], a.start[b + 1], a.tokens);
    raw = a.len[b];
    first = t.first, count = t.count;
    len = min(max(raw, 0), most);
  };
  auto is_big = [&] { return (long long)count * p.group >= p.big; };
  auto steps_of = [&](int tokens, int chunk) {
    const int span = g.window > 0 ? (int)min((long long)len, g.window + tokens + 14) : len;
    return max(1, (span + chunk - 1) / chunk);
  };
  auto cut = [&] {
    const bool mine_too = (on && is_big()) == LAST;
    items = mine_too ? (count + p.tile_tokens - 1) / p.tile_tokens * heads : 0;
    steps = steps_of(p.tile_tokens, p.chunk);
  };
  auto of = [&](int b) {
    load(b);
    cut();
  };
  auto total_of = [&](float v) {
#pragma unroll
    for (int i = 1; i < 64; i *= 2) v += __shfl_xor(v, i);
    return v;
  };
  // the totals, in f32: they only have to be the same for all waves
  load(lane);
  if (p.big < kNever) {
    float tiles = 0.0f;
    for (int b0 = 0; b0 < a.batch; b0 += 64) {
      if (a.batch > 64) load(b0 + lane);
      const int n = is_big() ? (count + p.big_tokens - 1) / p.big_tokens * a.kv_heads : 0;
      tiles += total_of((float)n * (float)steps_of(p.big_tokens, 64));
    }
    on = tiles >= p.big_steps;
  }
  cut();
  float all = 0.0f;
  for (int b0 = 0; b0 < a.batch; b0 += 64) {
    if (a.batch > 64) of(b0 + lane);
    all += total_of((float)items * (float)steps);
  }
  const int length = max(p.least, (int)fminf(ceilf(all / (float)p.waves), 1e9f));
  auto parts = [&] { return steps < p.whole * length ? 1 : (steps - 1) / length + 1; };
  *joined = 0;
  if (mine == 0) {
    for (int b0 = 0; b0 < a.batch; b0 += 64) {
      if (a.batch > 64) of(b0 + lane);
      *joined += __builtin_amdgcn_readlane(sums_upto(parts() > 1 ? items : 0), 63);
    }
    if (a.batch > 64) of(lane);
  }
  if (LAST) {
    int splits = 0;
    for (int b0 = 0; b0 < a.batch; b0 += 64) {
      if (a.batch > 64) of(b0 + lane);
      splits += __builtin_amdgcn_readlane(sums_upto(items * parts()), 63);
    }
    mine = splits - 1 - mine;
    if (mine < 0) return false;
  }
  int before = 0, items_before = 0, slots_before = 0;
  for (int b0 = 0; b0 < a.batch && before <= mine; b0 += 64) {
    if (a.batch > 64) of(b0 + lane);
    const int n = parts(), here = items * n, several = n > 1 ? items : 0;
    const int upto = sums_upto(here), items_upto = sums_upto(several), slots_upto = sums_upto(several * n);
    const unsigned long long hit = __ballot(mine >= before + upto - here && mine < before + upto);
    if (hit) {
      const int src = __ffsll(hit) - 1;
      s->of = __builtin_amdgcn_readlane(n, src);
      const int at = mine - before - __builtin_amdgcn_readlane(upto - here, src);
      // the splits of a kv head side by side: on one XCD, where there are eight
      const int each = __builtin_amdgcn_readlane(items, src);
      s->index = at / each;
      const int item = at - s->index * each, tile = item / heads, hh = item - tile * heads;
      s->item = items_before + __builtin_amdgcn_readlane(items_upto - several, src) + item;
      s->slot = slots_before + __builtin_amdgcn_readlane(slots_upto - several * n, src) + item * s->of;
      s->seq = b0 + src;
      s->kv_head = hh / p.head_tiles;
      s->head = s->kv_head * p.group + (hh - s->kv_head * p.head_tiles) * 16;
      const int skip = tile * p.tile_tokens, whole = __builtin_amdgcn_readlane(count, src);
      s->token = __builtin_amdgcn_readlane(first, src) + skip;
      s->count = min(whole - skip, p.tile_tokens);
      s->len = __builtin_amdgcn_readlane(len, src);
      // the raw length places the tokens, whatever the table holds
      s->pos = (long long)__builtin_amdgcn_readlane(raw, src) - whole + skip;
      s->first = s->index * length;
      const int steps_all = __builtin_amdgcn_readlane(steps, src);
      s->steps = s->of == 1 ? steps_all : min(length, steps_all - s->first);
      return true;
    }
    before += __builtin_amdgcn_readlane(upto, 63);
    items_before += __builtin_amdgcn_readlane(items_upto, 63);
    slots_before += __builtin_amdgcn_readlane(slots_upto, 63);
  }
  return false;
}

// What the join needs to know: how many items have several splits, from split
// 0, and of each of them, from its first.
__device__ __forceinline__ void note_item(const SplitArgs& p, int id, const Split& s, bool have, int joined) {
  if (!p.slots) return;
  if (id == 0) p.table[0].x = joined;
  if (have && s.of > 1 && s.index == 0 && (uint32_t)s.item < (uint32_t)p.joined)
    p.table[1 + s.item] = make_int4(s.slot, s.of | s.count << 24, s.token, s.head);
}

// A value that all lanes have, in a scalar register (64-bit comparisons leave
// vector ones).
__device__ __forceinline__ int shared(int v) { return __builtin_amdgcn_readfirstlane(v); }

__device__ __forceinline__ float max_of_rows(float v) {  // over the four lanes of a column
  v = fmaxf(v, __shfl_xor(v, 16));
  return fmaxf(v, __shfl_xor(v, 32));
}
__device__ __forceinline__ float sum_of_rows(float v) {
  v += __shfl_xor(v, 16);
  return v + __shfl_xor(v, 32);
}

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));

template <int J>
__device__ __forceinline__ h16x2 mx_pair(uint32_t w, float scale) {
  return __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, scale, J);
}
__device__ __forceinline__ f16x8 mx_eight(uint32_t w, float scale) {
  const h16x2 a = mx_pair<0>(w, scale), b = mx_pair<1>(w, scale), c = mx_pair<2>(w, scale), d = mx_pair<3>(w, scale);
  return f16x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// A lane's quarter of a row: D / 4 elements, their words and scale bytes.  The
// scales come in the 32 bits that hold them, and ready() takes them out where
// the piece is used: done with the load, it would wait for it.
template <int D>
struct Piece {
  uint32_t w[D / 32];
  uint32_t s;  // D / 128 bytes, or the one the piece is half of
  __device__ __forceinline__ void load(const uint32_t* words, const uint8_t* scales, size_t row, int quarter) {
    const uint32_t* p = words + row * (D / 8) + quarter * (D / 32);
    if constexpr (D == 64) {
      const uint2 v = *(const uint2*)p;
      w[0] = v.x, w[1] = v.y;
      s = ((const uint32_t*)scales)[row / 2];
    } else if constexpr (D == 128) {
      const uint4 v = *(const uint4*)p;
      w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
      s = ((const uint32_t*)scales)[row];
    } else {
      const uint4 v = *(const uint4*)p, u = *(const uint4*)(p + 4);
      w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
      w[4] = u.x, w[5] = u.y, w[6] = u.z, w[7] = u.w;
      s = ((const uint32_t*)scales)[row * 2 + (quarter >> 1)];
    }
  }
  __device__ __forceinline__ void ready(int row, int quarter) {  // row: its last bit
    if constexpr (D == 64) s = s >> ((row & 1) * 16 + (quarter >> 1) * 8) & 255u;
    if constexpr (D == 128) s = s >> (quarter * 8) & 255u;
    if constexpr (D == 256) s = s >> ((quarter & 1) * 16) & 0xFFFFu;
  }
  __device__ __forceinline__ float scale(int word) const {
    return mx_scale(D == 256 && word >= 4 ? s >> 8 : D == 256 ? s & 255u : s);
  }
  __device__ __forceinline__ f16x8 eight(int word) const { return mx_eight(w[word], scale(word)); }
  // The piece's blocks that are NaN, or whose factor passes f16, as bits of the
  // row's blocks.
  static __device__ __forceinline__ bool bad(uint32_t byte) { return byte > 127u + 13u; }
  __device__ __forceinline__ uint32_t nan_bits(int quarter) const {
    if constexpr (D == 64) return bad(s) ? 1u << (quarter >> 1) : 0u;
    if constexpr (D == 128) return bad(s) ? 1u << quarter : 0u;
    return (bad(s & 255u) ? 1u << (2 * quarter) : 0u) | (bad(s >> 8) ? 2u << (2 * quarter) : 0u);
  }
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int i = 0; i < D / 32; ++i) w[i] = 0;
    s = D == 256 ? 0x7F7Fu : 127u;
  }
  __device__ __forceinline__ void clear_nan() {
    if constexpr (D == 256) {
      if (bad(s & 255u)) w[0] = w[1] = w[2] = w[3] = 0, s = (s & 0xFF00u) | 127u;
      if (bad(s >> 8)) w[4] = w[5] = w[6] = w[7] = 0, s = (s & 255u) | 0x7F00u;
    } else if (bad(s)) {
      clear();
    }
  }
};

// Attention of one tile over one split of its keys, by one wave.
//
// S^T = K Q^T on 16 x 16 x 32 matrix instructions: a lane's A operand is a
// quarter of one key's row (a whole MXFP4 block at d = 128, one scale), its B
// operand the same quarter of a query's; the order in which the products
// take the row's elements is the lanes', the same on both sides.  The
// result leaves a lane four keys of one query, and two such tiles are the B
// operand of O^T += V^T P^T as they stand, if the A operand takes the keys
// in that order: values go through LDS as f16 rows and come back transposed,
// four keys a read.  The running maximum moves only when a score passes it by
// 2^8, so that most steps leave the sums as they are.
//
// Each p is rounded to f16, the matrix instruction's type: 2^-11 of it, where the
// cache's own rounding of a value is 2^-3.  p in two halves would take the second
// product twice.  The sum of p stays f32, of p before it is rounded.
constexpr int kChunk = 64;  // keys a step
// An exponent is score * scale - ref in one rounding, ref being the reference's
// own product, rounded by up to 2^-24 of it.  Beyond kFar that is more than the
// exponentials' own error (and from 2^25 on whole powers of two, up to infinite
// or vanishing ones): scores are taken relative to the reference first there.
constexpr float kFar = 1024.0f;
// A wave's accesses of its own LDS before here go before those behind.
__device__ __forceinline__ void own_lds() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}
constexpr int split_row(int d) { return d * 2 + 32; }  // bytes in LDS: four rows side by side meet no bank twice
// W > 1: the W waves of a workgroup share the item's keys, and their sums meet
// in LDS (`met`: their statistics).
template <int D, int W = 1>
__device__ __forceinline__ bool attend_split(const KvArgs& a, const AttnArgs& g, const SplitArgs& p, int id, uint8_t* vt,
                                             int wave = 0, float2* met = nullptr) {
  constexpr int kRow = split_row(D);
  const int lane = threadIdx.x & 63, col = lane & 15, quad = lane >> 4;
  Split s;
  int joined;
  const bool have = plan<false>(a, g, p, id, &s, &joined);
  if (lane == 0) note_item(p, id, s, have, joined);
  if (!have) return false;
  if constexpr (W > 1) {
    const int each = (s.steps + W - 1) / W;
    s.first = wave * each;
    s.steps = min(each, s.steps - s.first);
  }
  // this lane's query
  const int within = p.tile_tokens > 1 ? col / p.group : 0;
  const int head = s.head + (p.tile_tokens > 1 ? col - within * p.group : col);
  const bool real = within < s.count && (p.tile_tokens > 1 ? col < p.tile_tokens * p.group
                                                           : head < (s.kv_head + 1) * p.group);
  const long long pos = s.pos + within;
  const int hi = !real ? 0 : (int)(g.causal ? max(0ll, min(s.len, pos + 1)) : s.len);
  const int lo = !real || g.window <= 0 ? 0 : (int)max(0ll, pos - g.window + 1);
  const long long last = s.pos + s.count - 1;
  const int most = shared((int)(g.causal ? max(0ll, min(s.len, last + 1)) : s.len));  // keys that some row sees: [from, most)
  const int from = shared(g.window > 0 ? (int)min((long long)most, max(0ll, s.pos - g.window + 1)) : 0);
  const int every = shared((int)(g.causal ? max(0ll, min(s.len, s.pos + 1)) : s.len));  // that all rows see, up to here
  const int all_from = shared(g.window > 0 ? (int)max(0ll, last - g.window + 1) : 0);
  f16x8 q[D / 32];
  {
    const uint16_t* src = g.q + (size_t)(s.token + within) * g.q_stride + g.q_off + (size_t)head * D + quad * (D / 4);
#pragma unroll
    for (int i = 0; i < D / 32; ++i) {
      if (real) {
        const Loose<uint16_t, 8> v = load_loose<uint16_t, 8>(src + i * 8);
#pragma unroll
        for (int e = 0; e < 8; ++e)
          q[i][e] = __builtin_bit_cast(_Float16, (uint16_t)(g.negate ? v.v[e] ^ 0x8000u : v.v[e]));
      } else {
        q[i] = f16x8{};
      }
    }
  }
  f32x4 o[D / 16] = {};
  float m = -INFINITY, l = 0.0f;  // the scores' reference (unscaled), the sum over this lane's keys
  uint32_t nan_blocks = 0;
  const int j0 = (from & ~15) + s.first * kChunk;
  const int steps = min(s.steps, (most - j0 + kChunk - 1) / kChunk);
  const int32_t* table = a.table + (size_t)s.seq * a.max_pages;
  const int mask = (1 << a.page_shift) - 1;
  int pages = -1;
  Piece<D> k[4], v[4];
  uint32_t paged = 0;  // tiles of 16 keys that lie on a page of the cache
  auto load = [&](int step, Piece<D>* kk, Piece<D>* vv) {
    uint32_t ok = 0;
    if ((step & 15) == 0) {  // the pages of 64 tiles, one a lane
      const long long j = (long long)j0 + (step * 4 + lane) * 16;
      pages = j < most ? table[j >> a.page_shift] : -1;
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int j = j0 + step * kChunk + u * 16;
      int page = __builtin_amdgcn_readlane(pages, (step * 4 + u) & 63);
      if ((uint32_t)page < (uint32_t)a.num_pages)
        ok |= 1u << u;
      else
        page = 0;
      const size_t row = (((size_t)page * a.kv_heads + s.kv_head) << a.page_shift) + (j & mask);
      kk[u].load(a.kc, a.ks, row + col, quad);
      vv[u].load(a.vc, a.vs, row + (lane >> 2), lane & 3);
    }
    return ok;
  };
  if (steps > 0) paged = load(0, k, v);
  for (int step = 0; step < steps; ++step) {
    Piece<D> kn[4], vn[4];
    uint32_t next = 0;
    if (step + 1 < steps) next = load(step + 1, kn, vn);
    const int j = j0 + step * kChunk;
#pragma unroll
    for (int u = 0; u < 4; ++u) k[u].ready(col, quad), v[u].ready(lane >> 2, lane & 3);
    f32x4 t[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      t[u] = f32x4{};
#pragma unroll
      for (int i = 0; i < D / 32; ++i) t[u] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k[u].eight(i), q[i], t[u], 0, 0, 0);
    }
    if (paged != 15u || j + kChunk > every || j < all_from) {  // the same for the whole wave
      uint32_t see = 0;
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const bool there = paged >> u & 1;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int key = j + u * 16 + quad * 4 + r;
          const bool yes = there && key < hi && key >= lo;
          see |= (uint32_t)yes << (u * 4 + r);
          t[u][r] = yes ? t[u][r] : -INFINITY;
        }
        // values that no row sees must not reach the sums, whatever they hold
        const int key = j + u * 16 + (lane >> 2);
        if (!there || key >= most || key < from) v[u].clear();
        // nor those that only some see, if they are NaN
        if (s.count > 1) {
          const uint32_t own = v[u].nan_bits(lane & 3);
          if (__ballot(own != 0)) {
            uint32_t row = own | __shfl_xor(own, 1);
            row |= __shfl_xor(row, 2);
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              const uint32_t of = __shfl(row, (quad * 4 + r) * 4);
              if (see >> (u * 4 + r) & 1) nan_blocks |= of;
            }
            if (own) v[u].clear_nan();
          }
        }
      }
    }
    float top = -INFINITY;
#pragma unroll
    for (int u = 0; u < 4; ++u) top = fmaxf(top, fmaxf(fmaxf(t[u][0], t[u][1]), fmaxf(t[u][2], t[u][3])));
    if (__ballot(m == -INFINITY ? top > m : (top - m) * g.scale > 8.0f)) {
      const float now = fmaxf(m, max_of_rows(top));
      const float f = now == m ? 1.0f : m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f((m - now) * g.scale);
      l *= f;
#pragma unroll
      for (int i = 0; i < D / 16; ++i) o[i] *= f;
      m = now;
    }
    // 2^6 times: a p of 2^-20 of the largest is still a normal f16 number
    float ref = (m == -INFINITY ? 0.0f : m * g.scale) - 6.0f;
    if (__ballot(fabsf(ref) > kFar)) {
      const float from_m = m == -INFINITY ? 0.0f : m;
#pragma unroll
      for (int u = 0; u < 4; ++u)
#pragma unroll
        for (int r = 0; r < 4; ++r) t[u][r] -= from_m;
      ref = -6.0f;
    }
    f16x8 pr[2];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const float e = __builtin_amdgcn_exp2f(fmaf(t[u][r], g.scale, -ref));  // 0 for a masked one
        l += e;
        pr[u >> 1][(u & 1) * 4 + r] = (_Float16)e;
      }
    }
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      own_lds();
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        f16x8* dst = (f16x8*)(vt + (u * 16 + (lane >> 2)) * kRow + (lane & 3) * (D / 2));
#pragma unroll
        for (int i = 0; i < D / 32; ++i) dst[i] = v[half * 2 + u].eight(i);
      }
      own_lds();
#pragma unroll
      for (int i = 0; i < D / 16; ++i) {
        // a group of 16 lanes reads 4 keys x 16 elements; lane e of it gets element e of the four
        typedef __attribute__((address_space(3))) s16x4* Lds;
        const uint8_t* src = vt + (quad * 4 + (col >> 2)) * kRow + i * 32 + (col & 3) * 8;
        const s16x4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((Lds)src);
        const s16x4 y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((Lds)(src + 16 * kRow));
        typedef short s16x8 __attribute__((ext_vector_type(8)));
        const s16x8 xy = {x[0], x[1], x[2], x[3], y[0], y[1], y[2], y[3]};
        o[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, xy), pr[half], o[i], 0, 0, 0);
      }
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) k[u] = kn[u], v[u] = vn[u];
    paged = next;
  }
  l = sum_of_rows(l);
  nan_blocks |= __shfl_xor(nan_blocks, 16);
  nan_blocks |= __shfl_xor(nan_blocks, 32);
  if (__ballot(nan_blocks != 0)) {
#pragma unroll
    for (int i = 0; i < D / 16; ++i)
      if (nan_blocks >> (i / 2) & 1) o[i] = f32x4{NAN, NAN, NAN, NAN};
  }
  if constexpr (W > 1) {
    own_lds();
#pragma unroll
    for (int i = 0; i < D / 16; ++i) *(f32x4*)((float*)vt + col * D + i * 16 + quad * 4) = o[i];
    if (quad == 0) met[wave * 16 + col] = make_float2(m, l);
    __syncthreads();
    const uint8_t* first = vt - wave * 32 * kRow;
    for (int t = threadIdx.x; t < 16 * (D / 4); t += W * 64) {
      const int r = t / (D / 4), c = t % (D / 4), in = p.tile_tokens > 1 ? r / p.group : 0, h = s.head + r - in * p.group;
      if (in >= s.count || h >= (s.kv_head + 1) * p.group) continue;
      float top = -INFINITY, sum = 0.0f;
#pragma unroll
      for (int w = 0; w < W; ++w) top = fmaxf(top, met[w * 16 + r].x);
      top = top == -INFINITY ? 0.0f : top;
      f32x4 y = {};
#pragma unroll
      for (int w = 0; w < W; ++w) {
        const float2 st = met[w * 16 + r];
        const float weight = __builtin_amdgcn_exp2f((st.x - top) * g.scale);
        sum = fmaf(weight, st.y, sum);
        y += weight * *(const f32x4*)((const float*)(first + w * 32 * kRow) + r * D + c * 4);
      }
      const float f = sum == 0.0f ? 0.0f : 1.0f / sum;
      ushort4 n;
      n.x = narrow<uint16_t>(y[0] * f), n.y = narrow<uint16_t>(y[1] * f);
      n.z = narrow<uint16_t>(y[2] * f), n.w = narrow<uint16_t>(y[3] * f);
      *(ushort4*)(g.y + ((size_t)(s.token + in) * g.heads + h) * D + c * 4) = n;
    }
    return true;
  }
  if (s.of == 1) {
    if (!real) return true;
    uint16_t* y = g.y + ((size_t)(s.token + within) * g.heads + head) * D + quad * 4;
    const float f = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
    for (int i = 0; i < D / 16; ++i) {
      ushort4 h;
      h.x = narrow<uint16_t>(o[i][0] * f), h.y = narrow<uint16_t>(o[i][1] * f);
      h.z = narrow<uint16_t>(o[i][2] * f), h.w = narrow<uint16_t>(o[i][3] * f);
      *(ushort4*)(y + i * 16) = h;
    }
    return true;
  }
  const int slot = s.slot + s.index;
  if (!real || (uint32_t)slot >= (uint32_t)p.slots) return true;
  float* out = p.sums + ((size_t)slot * p.rows + col) * D + quad * 4;
#pragma unroll
  for (int i = 0; i < D / 16; ++i) *(f32x4*)(out + i * 16) = o[i];
  if (quad == 0) p.stats[(size_t)slot * p.rows + col] = make_float2(m, l);
  return true;
}

template <int D>
__global__ __launch_bounds__(64) void attention_split_kernel(KvArgs a, AttnArgs g, SplitArgs p) {
  __shared__ __align__(16) uint8_t vt[32 * split_row(D)];
  attend_split<D>(a, g, p, blockIdx.x, vt);
}

// Few steps: a workgroup takes an item whole, and nothing is joined by another
// launch.
constexpr int group_waves(int d) { return d == 256 ? 4 : 8; }
template <int D>
__global__ __launch_bounds__(64 * group_waves(D)) void attention_group_kernel(KvArgs a, AttnArgs g, SplitArgs p) {
  constexpr int W = group_waves(D);
  extern __shared__ __align__(16) uint8_t group_lds[];
  __shared__ float2 met[W * 16];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  attend_split<D, W>(a, g, p, blockIdx.x, group_lds + wave * 32 * split_row(D), wave, met);
}

constexpr int kJoinSplits = 1024;

// Joins the splits of an item: a workgroup for some of its rows, one after the
// other, D / 4 threads a split, so that J = 512 reads 8 to 32 splits at a time;
// the threads' sums meet in LDS in a fixed order.
template <int D, int J>
__device__ __forceinline__ void join_rows(const AttnArgs& g, const SplitArgs& p, int4 item, int from) {
  constexpr int kWide = J / (D / 4);  // splits at a time
  __shared__ float weight[kJoinSplits], part[2][J / 64];
  __shared__ f32x4 sums[J];
  const int tid = threadIdx.x;
  const int splits = item.y & 0xFFFFFF, count = (int)((uint32_t)item.y >> 24);
  if (!entry_fits(item.x, splits, item.z, item.w, p.slots, g.tokens, g.heads)) return;
  for (int col = from; col < p.rows; col += gridDim.y) {
    const int within = p.tile_tokens > 1 ? col / p.group : 0, head = item.w + col - within * p.group;
    if (within >= count || head >= (item.w / p.group + 1) * p.group) return;  // nor are the rows behind it
    if (item.z >= g.tokens - within || head >= g.heads) return;
    const float2* stats = p.stats + (size_t)item.x * p.rows + col;
    float m = -INFINITY;
    for (int i = tid; i < splits; i += J) m = fmaxf(m, stats[(size_t)i * p.rows].x);
    for (int i = 1; i < 64; i *= 2) m = fmaxf(m, __shfl_xor(m, i));
    __syncthreads();  // the row before is done
    if ((tid & 63) == 0) part[0][tid >> 6] = m;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < J / 64; ++i) m = fmaxf(m, part[0][i]);
    const float ref = m == -INFINITY ? 0.0f : m;
    const int at = tid % (D / 4), lane = tid / (D / 4);
    const float* src = p.sums + ((size_t)item.x * p.rows + col) * D + at * 4;
    f32x4 o = {};
    float l = 0.0f;
    for (int i0 = 0; i0 < splits; i0 += kJoinSplits) {
      const int n = min(kJoinSplits, splits - i0);
      __syncthreads();
      for (int i = tid; i < n; i += J) {
        const float2 st = stats[(size_t)(i0 + i) * p.rows];
        const float w = __builtin_amdgcn_exp2f((st.x - ref) * g.scale);
        weight[i] = w;
        l = fmaf(w, st.y, l);
      }
      __syncthreads();
#pragma unroll 4
      for (int i = lane; i < n; i += kWide) o += weight[i] * *(const f32x4*)(src + (size_t)(i0 + i) * p.rows * D);
    }
    for (int i = 1; i < 64; i *= 2) l += __shfl_xor(l, i);
    if ((tid & 63) == 0) part[1][tid >> 6] = l;
    sums[tid] = o;
    __syncthreads();
    if (tid >= D / 4) continue;
    l = part[1][0];
#pragma unroll
    for (int i = 1; i < J / 64; ++i) l += part[1][i];
#pragma unroll
    for (int i = 1; i < kWide; ++i) o += sums[i * (D / 4) + tid];
    const float f = l == 0.0f ? 0.0f : 1.0f / l;
    ushort4 h;
    h.x = narrow<uint16_t>(o[0] * f), h.y = narrow<uint16_t>(o[1] * f);
    h.z = narrow<uint16_t>(o[2] * f), h.w = narrow<uint16_t>(o[3] * f);
    *(ushort4*)(g.y + ((size_t)(item.z + within) * g.heads + head) * D + tid * 4) = h;
  }
}

template <int D, int J>
__global__ __launch_bounds__(J) void attention_join_kernel(AttnArgs g, SplitArgs p) {
  // the entry need not wait for their number
  const int4 item = p.table[1 + blockIdx.x];
  if ((int)blockIdx.x < p.table[0].x) join_rows<D, J>(g, p, item, blockIdx.y);
}

// Those of both forms.
template <int D>
__global__ __launch_bounds__(64) void attention_join_both_kernel(AttnArgs g, SplitArgs one, SplitArgs two) {
  const int n_one = one.slots ? min(one.table[0].x, one.joined) : 0, n_two = two.slots ? min(two.table[0].x, two.joined) : 0;
  for (int i = blockIdx.x; i < n_one; i += gridDim.x) join_rows<D, 64>(g, one, one.table[1 + i], blockIdx.y);
  for (int i = blockIdx.x; i < n_two; i += gridDim.x) join_rows<D, 64>(g, two, two.table[1 + i], blockIdx.y);
}

// --- many new tokens ---------------------------------------------------------------

typedef float f32x16 __attribute__((ext_vector_type(16)));

constexpr int tile_keys(int d) { return d == 256 ? 32 : 64; }  // keys a step

// All waves' accesses of LDS before here go before those behind; loads of global
// memory stay in flight (__syncthreads would wait for them).
__device__ __forceinline__ void lds_barrier() {
  __builtin_amdgcn_s_waitcnt(0xC07F);  // LDS alone
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// A tile of up to 128 rows (new tokens of a sequence x heads of a kv head) over
// all of its keys or a split of them, 32 rows a wave.
//
// KT keys a step: a thread widens a quarter of a key's and of a value's row to
// f16 (their packed form was loaded a step before) and writes it to LDS, where
// the four waves read it: the conversion, not the bytes, would bound the
// kernel if each wave made its own.  S^T = K Q^T and O^T += V^T P^T on
// 32 x 32 x 16 matrix instructions: the first's result leaves a lane keys of
// one row that are the second's B operand as they stand, if V^T takes the keys
// in that order, which transposing reads of LDS give it.  Two workgroups fit a
// CU up to d = 128, so that one's exponentials run beside the other's products.
//
// 4,096 causal tokens of 32 heads over 8 kv heads, d = 128: 159 us, 865 TFLOP/s.
// The products take a third of that and the vector instructions (exponentials,
// conversions) half; two waves a SIMD do not hide all of either.
//
// Sequences of few rows, whose splits are a wave's, take the workgroups behind
// the tiles'.
template <int D>
__global__ __launch_bounds__(256, D == 256 ? 1 : 2) void attention_tile_kernel(KvArgs a, AttnArgs g, SplitArgs p,
                                                                                SplitArgs few) {
  constexpr int KT = tile_keys(D);
  // Bytes of a row in LDS, such that lanes that go together meet no bank twice:
  // a key's with 16 behind it; a value's 16-byte pieces stand at their index
  // xor 5 s, for 4 rows beside each other that are read by 64 bytes each and
  // written by 16.
  constexpr int kKeyRow = D * 2 + 16, kValueRow = D * 2;
  constexpr int kBuffer = KT * (kKeyRow + kValueRow), kReads = 3, kPairs = 4;
  auto turned = [](int row) { return 5 * (D == 64 ? row >> 1 & 1 : row & 3); };
  extern __shared__ __align__(16) uint8_t lds[];
  __shared__ uint32_t nan_lds[2][KT];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int row = lane & 31, half = lane >> 5;
  if ((int)blockIdx.x >= p.splits) {  // sequences of few rows
    for (int id = ((int)blockIdx.x - p.splits) * 4 + wave; id < few.splits; id += ((int)gridDim.x - p.splits) * 4)
      if (!attend_split<D>(a, g, few, id, lds + wave * 32 * split_row(D))) break;
    return;
  }
  // a sequence's last tiles, which see the most keys, go first
  Split s;
  int joined;
  const bool have = plan<true>(a, g, p, blockIdx.x, &s, &joined);
  if (tid == 0) note_item(p, blockIdx.x, s, have, joined);
  if (!have) return;
  const int kv_head = s.kv_head, seq = s.seq, start = s.token;
  const long long len = s.len, pos0 = s.pos, pos1 = pos0 + s.count - 1;
  // this lane's row
  const int r = wave * 32 + row, within = r / p.group, head = s.head + r - within * p.group;
  const bool real = within < s.count;
  const int token = start + within;
  const long long pos = pos0 + within;
  const int hi = !real ? 0 : (int)(g.causal ? max(0ll, min(len, pos + 1)) : len);
  const int lo = !real || g.window <= 0 ? 0 : (int)max(0ll, pos - g.window + 1);
  const int most = shared((int)(g.causal ? max(0ll, min(len, pos1 + 1)) : len));  // keys that some row sees: [from, most)
  const int from = shared(g.window > 0 ? (int)min((long long)most, max(0ll, pos0 - g.window + 1)) : 0);
  const int every = shared((int)(g.causal ? max(0ll, min(len, pos0 + 1)) : len));  // that all rows see, up to here
  const int all_from = shared(g.window > 0 ? (int)max(0ll, pos1 - g.window + 1) : 0);
  f16x8 q[D / 16];
  {
    const uint16_t* src = g.q + (size_t)(real ? token : start) * g.q_stride + g.q_off + (size_t)head * D + half * 8;
#pragma unroll
    for (int i = 0; i < D / 16; ++i) {
      q[i] = f16x8{};
      if (real) {
        const Loose<uint16_t, 8> v = load_loose<uint16_t, 8>(src + i * 16);
#pragma unroll
        for (int e = 0; e < 8; ++e)
          q[i][e] = __builtin_bit_cast(_Float16, (uint16_t)(g.negate ? v.v[e] ^ 0x8000u : v.v[e]));
      }
    }
  }
  f32x16 o[D / 32] = {};
  float m = -INFINITY, l = 0.0f, l1 = 0.0f;
  uint32_t nan_blocks = 0;
  const int j0 = shared((from & ~15) + s.first * KT), steps = shared(min(s.steps, (most - j0 + KT - 1) / KT));
  const int32_t* table = a.table + (size_t)seq * a.max_pages;
  const int mask = (1 << a.page_shift) - 1;
  // the page of key `lane` of a step, or -1
  auto page_of = [&](int step) {
    const long long j = (long long)j0 + (long long)step * KT + lane;
    return lane < KT && j < most ? table[j >> a.page_shift] : -1;
  };
  auto on_page = [&](int page) { return (uint32_t)page < (uint32_t)a.num_pages; };
  // this thread's part of the widening: a quarter of one key's row
  const bool does_k = KT == 64 || wave < 2, does_v = KT == 64 || wave >= 2;
  const int key = (tid >> 2) % KT, quarter = tid & 3;
  Piece<D> k, v;
  auto row_of = [&](int step, int pages) {
    const int j = j0 + step * KT + key;
    int page = __shfl(pages, key);
    page = on_page(page) ? page : 0;  // a key on no page is seen by no row: any row's bytes will do
    return (((size_t)page * a.kv_heads + kv_head) << a.page_shift) + (j & mask);
  };
  // kept from being added to the four bases ahead of the loop, whose registers
  // would push others to memory
  auto anew = [](int v) {
    asm volatile("" : "+v"(v));
    return v;
  };
  auto fetch_k = [&](Piece<D>& to, int step, int pages) {
    const size_t at = row_of(step, pages);
    if (does_k) to.load(a.kc, a.ks, at, anew(quarter));
  };
  auto fetch_v = [&](int step, int pages) {
    const size_t at = row_of(step, pages);
    if (does_v) v.load(a.vc, a.vs, at, anew(quarter));
  };
  auto whole = [&](int step, unsigned long long there) {
    const int j = j0 + step * KT;
    return there == ~0ull >> (64 - KT) && j + KT <= every && j >= all_from;
  };
  // Values that no row sees must not reach the sums, whatever they hold, nor
  // those that only some see, if they are NaN.
  auto clean_v = [&](int step, unsigned long long there) {
    if (!does_v || whole(step, there)) return;
    const int j = j0 + step * KT + key;
    if (!(there >> key & 1) || j >= most || j < from) v.clear();
    const uint32_t own = v.nan_bits(quarter);
    uint32_t bits = own | __shfl_xor(own, 1);
    bits |= __shfl_xor(bits, 2);
    if (own) v.clear_nan();
    if (quarter == 0) nan_lds[step & 1][key] = bits;
  };
  auto widen_k = [&](const Piece<D>& piece, int step, int i) {
    if (does_k)
      *(f16x8*)(lds + (step & 1) * kBuffer + key * kKeyRow + quarter * (D / 2) + i * 16) = piece.eight(i);
  };
  auto widen_v = [&](int step, int i) {
    if (does_v)
      *(f16x8*)(lds + (step & 1) * kBuffer + KT * kKeyRow + key * kValueRow +
                (((quarter * (D / 32) + i) ^ turned(key)) * 16)) = v.eight(i);
  };
  // Scores of 32 keys, with other work beside each product.
  auto scores = [&](int step, int u, f32x16& t, auto beside) {
    const uint8_t* kb = lds + (step & 1) * kBuffer + (u * 32 + row) * kKeyRow + half * 16;
    f16x8 x[D / 16];
#pragma unroll
    for (int i = 0; i < kReads; ++i) x[i] = *(const f16x8*)(kb + i * 32);
    t = f32x16{};
#pragma unroll
    for (int i = 0; i < D / 16; ++i) {
      if (i + kReads < D / 16) x[i + kReads] = *(const f16x8*)(kb + (i + kReads) * 32);
      t = __builtin_amdgcn_mfma_f32_32x32x16_f16(x[i], q[i], t, 0, 0, 0);
      beside(i);
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  // a lane's place among the values: its row and, in it, piece and half, without
  // the part of the turn that goes over 64 bytes
  const int e16 = lane & 15, value_turn = turned(e16 >> 2) & 12;
  const int value_at = (4 * half + (e16 >> 2)) * kValueRow +
                       ((((lane >> 4) & 1) * 2 + ((e16 & 3) >> 1)) ^ (turned(e16 >> 2) & 3)) * 16 + (e16 & 1) * 8;
  // Step s's scores are formed a step ahead, beside the exponentials of the step
  // before: its keys are in LDS then, its values a step later.
  unsigned long long there = 0, there1 = 0, there2 = 0;
  int pages_v = -1, pages_k = -1;
  f32x16 t[KT / 32];
  if (steps > 0) {
    const int pages0 = page_of(0), pages1 = page_of(1), pages2 = page_of(2);
    pages_k = page_of(3);
    there = __ballot(on_page(pages0)), there1 = __ballot(on_page(pages1)), there2 = __ballot(on_page(pages2));
    Piece<D> next;
    fetch_k(k, 0, pages0);
    fetch_v(0, pages0);
    if (steps > 1) fetch_k(next, 1, pages1);
    k.ready(key, quarter), v.ready(key, quarter);
    clean_v(0, there);
#pragma unroll
    for (int i = 0; i < D / 32; ++i) widen_k(k, 0, i), widen_v(0, i);
    if (steps > 1) {
      next.ready(key, quarter);
#pragma unroll
      for (int i = 0; i < D / 32; ++i) widen_k(next, 1, i);
      fetch_v(1, pages1);
    }
    if (steps > 2) fetch_k(k, 2, pages2);
    pages_v = pages2;
    __syncthreads();
#pragma unroll
    for (int u = 0; u < KT / 32; ++u) scores(0, u, t[u], [](int) {});
  }
  for (int step = 0; step < steps; ++step) {
    if (!whole(step, there)) {
      // this lane's keys are 8 (e / 4) + e % 4 of each 32, from `base` on
      const int base = j0 + step * KT + 4 * half;
      auto first = [](int n) { return n >= 64 ? ~0ull : (1ull << max(n, 0)) - 1; };
      const unsigned long long see = there >> (4 * half) & first(hi - base) & ~first(lo - base);
#pragma unroll
      for (int u = 0; u < KT / 32; ++u)
#pragma unroll
        for (int e = 0; e < 16; ++e) t[u][e] = see >> (u * 32 + 8 * (e / 4) + e % 4) & 1 ? t[u][e] : -INFINITY;
      const uint32_t any = lane < KT ? nan_lds[step & 1][lane] : 0u;
      if (__ballot(any != 0)) {
        const uint32_t* of = &nan_lds[step & 1][4 * half];
#pragma unroll
        for (int u = 0; u < KT / 32; ++u)
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            const int c = u * 32 + 8 * (e / 4) + e % 4;
            if (see >> c & 1) nan_blocks |= of[c];
          }
      }
    }
    float top = -INFINITY, top1 = -INFINITY;
#pragma unroll
    for (int u = 0; u < KT / 32; ++u)
#pragma unroll
      for (int e = 0; e < 16; e += 4)
        top = fmaxf(fmaxf(top, t[u][e]), t[u][e + 1]), top1 = fmaxf(fmaxf(top1, t[u][e + 2]), t[u][e + 3]);
    top = fmaxf(top, top1);
    if (__ballot(m == -INFINITY ? top > m : (top - m) * g.scale > 8.0f)) {
      const float now = fmaxf(m, fmaxf(top, __shfl_xor(top, 32)));
      const float f = now == m ? 1.0f : m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f((m - now) * g.scale);
      l *= f, l1 *= f;
#pragma unroll
      for (int i = 0; i < D / 32; ++i) o[i] *= f;
      m = now;
    }
    k.ready(key, quarter), v.ready(key, quarter);
    if (step + 1 < steps) clean_v(step + 1, there1);
    // 2^6 times: a p of 2^-20 of the largest is still a normal f16 number
    float ref = (m == -INFINITY ? 0.0f : m * g.scale) - 6.0f;
    if (__ballot(fabsf(ref) > kFar)) {
      const float from_m = m == -INFINITY ? 0.0f : m;
#pragma unroll
      for (int u = 0; u < KT / 32; ++u) t[u] -= from_m;
      ref = -6.0f;
    }
    f16x8 pr[KT / 16];
    // the matrix instructions of a wave go before the other's fetching and masks
    __builtin_amdgcn_s_setprio(1);
    auto exponential = [&](int u, int e) {
      const float x = __builtin_amdgcn_exp2f(fmaf(t[u][e], g.scale, -ref));  // 0 for a masked one
      (e & 1 ? l1 : l) += x;
      pr[u * 2 + e / 8][e % 8] = (_Float16)x;
      if (e & 1) asm volatile("" : "+v"(l), "+v"(l1));  // here, not all at the step's end
    };
#pragma unroll
    for (int e = 0; e < 16; ++e) exponential(0, e);
    __builtin_amdgcn_sched_barrier(0);
    // The next step's scores, behind the last one of what LDS holds (nothing
    // comes of it), take the registers that the exponentials leave.
#pragma unroll
    for (int u = 1; u < KT / 32; ++u)
      scores(step + 1, u - 1, t[u - 1], [&](int i) {
        constexpr int n = 16 / (D / 16);
#pragma unroll
        for (int e = 0; e < n; ++e) exponential(u, i * n + e);
      });
    // values and keys go into the places that the step before read last
    scores(step + 1, KT / 32 - 1, t[KT / 32 - 1], [&](int i) {
      if (i < D / 32)
        widen_v(step + 1, i);
      else
        widen_k(k, step + 2, i - D / 32);
    });
    // Four groups of 16 lanes read 4 keys x 16 elements each, and lane e of one
    // gets element e of the four.
    const uint8_t* vb = lds + (step & 1) * kBuffer + KT * kKeyRow + value_at;
    typedef short s16x8 __attribute__((ext_vector_type(8)));
    auto values = [&](int n) {
      typedef __attribute__((address_space(3))) s16x4* Lds;
      const int i = n / (KT / 16), u = n % (KT / 16);
      const uint8_t* src = vb + (((i * 4) ^ value_turn) * 16 + u * 16 * kValueRow);
      const s16x4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((Lds)src);
      const s16x4 y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((Lds)(src + 8 * kValueRow));
      return s16x8{x[0], x[1], x[2], x[3], y[0], y[1], y[2], y[3]};
    };
    constexpr int kProducts = D / 32 * (KT / 16);
    s16x8 pair[kProducts];
#pragma unroll
    for (int n = 0; n < kPairs; ++n) pair[n] = values(n);
#pragma unroll
    for (int n = 0; n < kProducts; ++n) {
      if (n + kPairs < kProducts) pair[n + kPairs] = values(n + kPairs);
      const int i = n / (KT / 16), u = n % (KT / 16);
      o[i] = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, pair[n]), pr[u], o[i], 0, 0, 0);
      __builtin_amdgcn_sched_barrier(0);
    }
    __builtin_amdgcn_s_setprio(0);
    if (step + 2 < steps) fetch_v(step + 2, pages_v);
    there = there1, there1 = there2;
    if (step + 3 < steps) {
      fetch_k(k, step + 3, pages_k);
      there2 = __ballot(on_page(pages_k));
      pages_v = pages_k;
      pages_k = page_of(step + 4);
    }
    lds_barrier();
  }
  l += l1;
  l += __shfl_xor(l, 32);
  nan_blocks |= __shfl_xor(nan_blocks, 32);
  if (!real) return;
  if (s.of > 1) {
    const int slot = s.slot + s.index;
    if ((uint32_t)slot >= (uint32_t)p.slots) return;
    float* out = p.sums + ((size_t)slot * p.rows + r) * D + half * 4;
#pragma unroll
    for (int i = 0; i < D / 32; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        f32x4 v = {o[i][e * 4], o[i][e * 4 + 1], o[i][e * 4 + 2], o[i][e * 4 + 3]};
        if (nan_blocks >> i & 1) v = f32x4{NAN, NAN, NAN, NAN};
        *(f32x4*)(out + i * 32 + e * 8) = v;
      }
    if (half == 0) p.stats[(size_t)slot * p.rows + r] = make_float2(m, l);
    return;
  }
  uint16_t* y = g.y + ((size_t)token * g.heads + head) * D + half * 4;
  const float f = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
  for (int i = 0; i < D / 32; ++i) {
    const float scale = nan_blocks >> i & 1 ? NAN : f;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      ushort4 h;
      h.x = narrow<uint16_t>(o[i][e * 4] * scale), h.y = narrow<uint16_t>(o[i][e * 4 + 1] * scale);
      h.z = narrow<uint16_t>(o[i][e * 4 + 2] * scale), h.w = narrow<uint16_t>(o[i][e * 4 + 3] * scale);
      *(ushort4*)(y + i * 32 + e * 8) = h;
    }
  }
}

}  // namespace

void launch_kv_append(hipStream_t st, const KvArgs& a, const void* k, size_t k_stride, size_t k_off, const void* v,
                      size_t v_stride, size_t v_off) {
  hipLaunchKernelGGL(kv_append_kernel, dim3((unsigned)a.tokens), dim3(256), 0, st, a, (const uint16_t*)k, k_stride,
                     k_off, (const uint16_t*)v, v_stride, v_off);
  DW_HIP(hipGetLastError());
}

namespace {

template <int D>
void launch_parts(hipStream_t st, const KvArgs& a, const AttnArgs& g, const AttnPlan& p) {
  if (p.tiles.splits) {
    constexpr int kLds = std::max(2 * tile_keys(D) * (D * 4 + 16), 4 * 32 * split_row(D));
    const unsigned grid = p.tiles.splits + std::min((p.few.splits + 3) / 4, 1024);
    hipLaunchKernelGGL(attention_tile_kernel<D>, dim3(grid), dim3(256), kLds, st, a, g, p.tiles, p.few);
  } else if (p.whole_groups) {
    constexpr int W = group_waves(D);
    hipLaunchKernelGGL(attention_group_kernel<D>, dim3((unsigned)p.few.items), dim3(64 * W), W * 32 * split_row(D), st, a,
                       g, p.few);
  } else {
    hipLaunchKernelGGL(attention_split_kernel<D>, dim3((unsigned)p.few.splits), dim3(64), 0, st, a, g, p.few);
  }
  if (!p.tiles.slots && !p.few.slots) return;
  // rows of few splits are many: a wave each then, or for eight of a tile's
  const dim3 grid(p.few.joined, p.few.rows);
  if (p.tiles.splits)
    hipLaunchKernelGGL(attention_join_both_kernel<D>, dim3(256, 16), dim3(64), 0, st, g, p.tiles, p.few);
  else if ((long long)a.tokens * g.heads > 512)
    hipLaunchKernelGGL((attention_join_kernel<D, 64>), grid, dim3(64), 0, st, g, p.few);
  else
    hipLaunchKernelGGL((attention_join_kernel<D, 512>), grid, dim3(512), 0, st, g, p.few);
}

}  // namespace

size_t attention_space(const KvArgs& a, const AttnArgs& g, AttnPlan* plan) {
  const int group = g.heads / a.kv_heads, longest = a.max_pages << a.page_shift;
  const long long rows = (long long)a.tokens * group;
  // Tiles of 128 rows do the work in half the time, tiles of 16 rows are done
  // sooner where there is little of it: 8 sequences of up to 128 new tokens
  // after 1,024 keys (32 heads over 8, d = 128) 51 us, 27 us in tiles of 16; 256
  // new tokens after 8,192 (64 tiles x 128 steps) 74 us, 86 us; 512 after 8,192 105
  // us, 162 us; 4,096 and as many keys 159 us, 315 us.
  // At d = 256 a CU holds four waves of them alone, and tiles pay sooner: 1,600 new
  // tokens of 7 heads over one after 1,200 keys 99 us, 145 us in tiles of 16; 512
  // after 1,200 65 us, 45 us, and alone 38 us, 26 us.
  //
  // The lengths are the device's: here and below, what the host chooses by is the
  // keys that the table has room for.
  constexpr int kBigRows = 128;
  const int big_steps = a.d == 256 ? 3000 : 6144;
  const bool tiles = group <= 128 && (double)rows * a.kv_heads / 128 * ((longest + 63) / 64) >= big_steps;
  auto fill = [&](SplitArgs* p, int most_rows, int chunk, int waves, int whole, int least) {
    p->big = tiles ? kBigRows : kNever;
    p->big_tokens = tiles ? 128 / group : 1;
    p->big_steps = big_steps;
    p->group = group;
    p->head_tiles = (group + most_rows - 1) / most_rows;
    p->tile_tokens = std::max(1, most_rows / group);
    p->rows = std::min(most_rows, group * p->tile_tokens);
    p->chunk = chunk;
    p->waves = waves;
    p->whole = whole;
    p->least = least;
    const long long heads = (long long)a.kv_heads * p->head_tiles;
    p->items = (int)(std::min<long long>(a.tokens, a.tokens / p->tile_tokens + (long long)a.batch) * heads);
    // 16 and 64: the steps' sum is rounded
    p->splits = p->items + waves + 16;
    p->slots = (longest + chunk - 1) / chunk > least ? 2 * waves + 64 : 0;
    p->joined = std::min(p->items, waves + 32);
  };
  const int many = a.d == 256 ? 1024 : 2048;  // waves that the chip holds at a time
  // A split of 128 rows leaves 64 KiB of sums at d = 128: items are split where
  // that shares them out over twice the workgroups or more (2 sequences of up to
  // 1,536 new tokens after 4,096 keys 140 us, 179 us with splits for every
  // uneven share), into eight steps or more.
  if (tiles) fill(&plan->tiles, 128, tile_keys(a.d), many / 4, 2, 8 * 64 / tile_keys(a.d));
  // A split of 16 rows takes two steps of 64 keys or more (one sequence of 1,024
  // keys 12.2 us so, 20.9 us in splits of eight).  Few steps need no second launch:
  // as many items as workgroups fit the chip take a workgroup each, a step a wave
  // (32 sequences of up to 500 keys 9.7 us, 15.9 us with a wave each; one of 500
  // 9.6 us, 12.3 us split and joined; two steps a wave at d = 128: one of 1,024
  // 12.0 us, 11.7 us split), and more items a wave each (64 of up to 500 16.4 us,
  // 17.5 us with a workgroup each).
  fill(&plan->few, 16, kChunk, many, 1, 2);
  const int steps = (longest + kChunk - 1) / kChunk, items = plan->few.items;
  plan->whole_groups = !tiles && steps > 1 && (a.d == 64 ? steps <= 16 && items <= 512
                                                         : steps <= group_waves(a.d) && items <= 256);
  if (plan->whole_groups || (steps <= 8 && items >= 256)) plan->few.least = steps, plan->few.slots = 0;
  size_t bytes = 0;
  int i = 0;
  for (const SplitArgs* p : {&plan->tiles, &plan->few}) {
    auto take = [&](size_t n) {
      const size_t at = bytes;
      bytes += (n + 255) / 256 * 256;
      return at;
    };
    size_t* at = plan->at[i++];
    if (!p->slots) continue;
    at[0] = take((size_t)p->slots * p->rows * a.d * 4);
    at[1] = take((size_t)p->slots * p->rows * 8);
    at[2] = take((size_t)(p->joined + 1) * 16);
  }
  return bytes;
}

void launch_attention(hipStream_t st, const KvArgs& a, const AttnArgs& g, AttnPlan p, void* space) {
  int i = 0;
  for (SplitArgs* s : {&p.tiles, &p.few}) {
    const size_t* at = p.at[i++];
    s->sums = (float*)((char*)space + at[0]);
    s->stats = (float2*)((char*)space + at[1]);
    s->table = (int4*)((char*)space + at[2]);
  }
  if (a.d == 64)
    launch_parts<64>(st, a, g, p);
  else if (a.d == 128)
    launch_parts<128>(st, a, g, p);
  else
    launch_parts<256>(st, a, g, p);
  DW_HIP(hipGetLastError());
}

}  // namespace dw
