// Attention over a cache of keys and values in MXFP4 pages, and what writes
// the cache.
//
// A page holds page_size rows of each kv head, [page][head][slot][d / 2]
// bytes and [page][head][slot][d / 32] scales: the rows are MXFP4 rows of d
// elements (mxfp4.h), so the cache's values can be read back as such rows.
#include <algorithm>
#include <type_traits>

#include "dw_common.h"
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
// element, written 17/32.  The scale is at least 2^-23, so that every value of
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

// A wave's share of the work: keys [begin, end) of a tile of up to 16 rows
// (new tokens of one sequence x heads of one kv head).
constexpr int kChunk = 64;  // keys a step

struct Split {
  int seq, token, count;  // the tile's first token and how many it has
  int kv_head, head;      // head: the tile's first
  int index, of;          // this split of the item's
  int first, chunks;      // steps before this split, and its own
  long long pos, len;     // position of the tile's first token, keys of the sequence
};

// Sums up to and with each lane, in the lanes' registers (six steps of data
// parallel primitives; each shuffle through LDS would cost several times one).
__device__ __forceinline__ int sums_upto(int v) {
  v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xF, 0xF, true);   // the lane one to the left in its row of 16
  v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xF, 0xF, true);   // two
  v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xF, 0xF, true);   // four
  v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xF, 0xF, true);   // eight
  v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xA, 0xF, false);  // the last of row 0 to row 1, of 2 to 3
  v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xC, 0xF, false);  // the last of row 1 to rows 2 and 3
  return v;
}

// Which split this wave has.  Every item (tile, kv head) of a sequence has
// the same number of steps; all steps over the waves wanted is a split's
// length, so that long and short sequences share the waves evenly whatever
// their lengths, which only the device knows.  One load a 64 sequences.
__device__ __forceinline__ bool plan(const KvArgs& a, const AttnArgs& g, const SplitArgs& p, int mine, Split* s) {
  const int lane = threadIdx.x & 63, heads = p.head_tiles * a.kv_heads;
  const int most = a.max_pages << a.page_shift;
  int first, items, steps, count, len, raw;
  auto of = [&](int b) {
    first = count = items = len = raw = 0;
    steps = 1;
    if (b >= a.batch) return;
    const int t0 = a.start[b], t1 = a.start[b + 1];
    raw = a.len[b];
    first = max(t0, 0);
    count = max(min(t1, a.tokens) - first, 0);
    len = min(max(raw, 0), most);
    items = (count + p.tile_tokens - 1) / p.tile_tokens * heads;
    const int span = g.window > 0 ? (int)min((long long)len, g.window + p.tile_tokens + 14) : len;
    steps = max(1, (span + kChunk - 1) / kChunk);
  };
  // the total, in f32: it only has to be the same for all waves
  float all = 0.0f;
  for (int b0 = 0; b0 < a.batch; b0 += 64) {
    of(b0 + lane);
    float v = (float)items * (float)steps;
#pragma unroll
    for (int i = 1; i < 64; i *= 2) v += __shfl_xor(v, i);
    all += v;
  }
  const int length = max(p.least, (int)fminf(ceilf(all / (float)p.waves), 1e9f));
  int before = 0;
  for (int b0 = 0; b0 < a.batch && before <= mine; b0 += 64) {
    if (a.batch > 64) of(b0 + lane);
    const int n = (steps - 1) / length + 1;
    const int upto = sums_upto(items * n), here = items * n;
    const unsigned long long hit = __ballot(mine >= before + upto - here && mine < before + upto);
    if (hit) {
      const int src = __ffsll(hit) - 1;
      s->of = __builtin_amdgcn_readlane(n, src);
      const int at = mine - before - __builtin_amdgcn_readlane(upto - here, src);
      const int item = at / s->of, tile = item / heads, hh = item - tile * heads;
      s->index = at - item * s->of;
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
      s->chunks = min(length, __builtin_amdgcn_readlane(steps, src) - s->first);
      return true;
    }
    before += __builtin_amdgcn_readlane(upto, 63);
  }
  return false;
}

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

// A lane's quarter of a row: D / 4 elements, their words and scale bytes.
template <int D>
struct Piece {
  uint32_t w[D / 32];
  uint32_t s;  // D / 128 bytes, or the one the piece is half of
  __device__ __forceinline__ void load(const uint32_t* words, const uint8_t* scales, size_t row, int quarter) {
    const uint32_t* p = words + row * (D / 8) + quarter * (D / 32);
    if constexpr (D == 64) {
      const uint2 v = *(const uint2*)p;
      w[0] = v.x, w[1] = v.y;
      s = scales[row * 2 + (quarter >> 1)];
    } else if constexpr (D == 128) {
      const uint4 v = *(const uint4*)p;
      w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
      s = scales[row * 4 + quarter];
    } else {
      const uint4 v = *(const uint4*)p, u = *(const uint4*)(p + 4);
      w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
      w[4] = u.x, w[5] = u.y, w[6] = u.z, w[7] = u.w;
      s = *(const uint16_t*)(scales + row * 8 + quarter * 2);
    }
  }
  __device__ __forceinline__ float scale(int word) const { return mx_scale(D == 256 && word >= 4 ? s >> 8 : D == 256 ? s & 255u : s); }
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
template <int D>
__global__ __launch_bounds__(64) void attention_split_kernel(KvArgs a, AttnArgs g, SplitArgs p) {
  constexpr int kRow = D * 2 + 32;  // bytes of a row in LDS: four rows side by side meet no bank twice
  __shared__ __align__(16) uint8_t vt[32 * kRow];
  const int lane = threadIdx.x, col = lane & 15, quad = lane >> 4;
  Split s;
  if (!plan(a, g, p, blockIdx.x, &s)) return;
  // this lane's query
  const int within = p.tile_tokens > 1 ? col / p.group : 0;
  const int head = s.head + (p.tile_tokens > 1 ? col - within * p.group : col);
  const bool real = within < s.count && (p.tile_tokens > 1 ? col < p.tile_tokens * p.group
                                                           : head < (s.kv_head + 1) * p.group);
  const long long pos = s.pos + within;
  const int hi = !real ? 0 : (int)(g.causal ? max(0ll, min(s.len, pos + 1)) : s.len);
  const int lo = !real || g.window <= 0 ? 0 : (int)max(0ll, pos - g.window + 1);
  const long long last = s.pos + s.count - 1;
  const int most = (int)(g.causal ? max(0ll, min(s.len, last + 1)) : s.len);  // keys that some row sees: [from, most)
  const int from = g.window > 0 ? (int)min((long long)most, max(0ll, s.pos - g.window + 1)) : 0;
  const int every = (int)(g.causal ? max(0ll, min(s.len, s.pos + 1)) : s.len);  // that all rows see, up to here
  const int all_from = g.window > 0 ? (int)max(0ll, last - g.window + 1) : 0;
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
  const int steps = min(s.chunks, (most - j0 + kChunk - 1) / kChunk);
  const int32_t* table = a.table + (size_t)s.seq * a.max_pages;
  const int mask = (1 << a.page_shift) - 1;
  int pages = -1;
  Piece<D> k[4], v[4];
  uint32_t have = 0;  // tiles of 16 keys that lie on a page of the cache
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
      if (page >= 0 && page < a.num_pages)
        ok |= 1u << u;
      else
        page = 0;
      const size_t row = (((size_t)page * a.kv_heads + s.kv_head) << a.page_shift) + (j & mask);
      kk[u].load(a.kc, a.ks, row + col, quad);
      vv[u].load(a.vc, a.vs, row + (lane >> 2), lane & 3);
    }
    return ok;
  };
  if (steps > 0) have = load(0, k, v);
  for (int step = 0; step < steps; ++step) {
    Piece<D> kn[4], vn[4];
    uint32_t next = 0;
    if (step + 1 < steps) next = load(step + 1, kn, vn);
    const int j = j0 + step * kChunk;
    f32x4 t[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      t[u] = f32x4{};
#pragma unroll
      for (int i = 0; i < D / 32; ++i) t[u] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k[u].eight(i), q[i], t[u], 0, 0, 0);
    }
    uint32_t see = 0xFFFFu;
    if (have != 15u || j + kChunk > every || j < all_from) {  // the same for the whole wave
      see = 0;
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const bool there = have >> u & 1;
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
    const float ref = (m == -INFINITY ? 0.0f : m * g.scale) - 6.0f;
    f16x8 pr[2];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        float e = __builtin_amdgcn_exp2f(fmaf(t[u][r], g.scale, -ref));
        e = see >> (u * 4 + r) & 1 ? e : 0.0f;
        l += e;
        pr[u >> 1][(u & 1) * 4 + r] = (_Float16)e;
      }
    }
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      __syncthreads();
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        f16x8* dst = (f16x8*)(vt + (u * 16 + (lane >> 2)) * kRow + (lane & 3) * (D / 2));
#pragma unroll
        for (int i = 0; i < D / 32; ++i) dst[i] = v[half * 2 + u].eight(i);
      }
      __syncthreads();
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
    have = next;
  }
  l = sum_of_rows(l);
  nan_blocks |= __shfl_xor(nan_blocks, 16);
  nan_blocks |= __shfl_xor(nan_blocks, 32);
  if (__ballot(nan_blocks != 0)) {
#pragma unroll
    for (int i = 0; i < D / 16; ++i)
      if (nan_blocks >> (i / 2) & 1) o[i] = f32x4{NAN, NAN, NAN, NAN};
  }
  if (s.index == 0 && lane == 0)
    p.items[(size_t)s.token * a.kv_heads * p.head_tiles + s.kv_head * p.head_tiles +
            (s.head - s.kv_head * p.group) / 16] = make_int2((int)blockIdx.x, s.of);
  if (s.of == 1) {
    if (!real) return;
    uint16_t* y = g.y + ((size_t)(s.token + within) * g.heads + head) * D + quad * 4;
    const float f = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
    for (int i = 0; i < D / 16; ++i) {
      ushort4 h;
      h.x = narrow<uint16_t>(o[i][0] * f), h.y = narrow<uint16_t>(o[i][1] * f);
      h.z = narrow<uint16_t>(o[i][2] * f), h.w = narrow<uint16_t>(o[i][3] * f);
      *(ushort4*)(y + i * 16) = h;
    }
    return;
  }
  if (!real) return;
  float* out = p.sums + ((size_t)blockIdx.x * p.rows + col) * D + quad * 4;
#pragma unroll
  for (int i = 0; i < D / 16; ++i) *(f32x4*)(out + i * 16) = o[i];
  if (quad == 0)
    p.stats[(size_t)blockIdx.x * p.rows + col] = make_float2(m == -INFINITY ? -INFINITY : m * g.scale, l);
}

constexpr int kJoinSplits = 1024;

// Joins the splits of an item, where it has several: a workgroup for each of
// its rows, D / 4 threads a split, so that J = 512 reads 8 to 32 splits at a time;
// the threads' sums meet in LDS in a fixed order.
template <int D, int J>
__global__ __launch_bounds__(J) void attention_join_kernel(KvArgs a, AttnArgs g, SplitArgs p) {
  constexpr int kWide = J / (D / 4);  // splits at a time
  __shared__ int found;
  __shared__ float weight[kJoinSplits], part[J / 64];
  __shared__ f32x4 sums[J];
  const int tid = threadIdx.x, t = blockIdx.x, hh = blockIdx.y, col = blockIdx.z;
  const int seq = sequence_of(a.start, a.batch, t, &found);
  if (seq >= a.batch || t < a.start[seq]) return;
  if ((t - max(a.start[seq], 0)) % p.tile_tokens) return;
  const int within = p.tile_tokens > 1 ? col / p.group : 0, kv_head = hh / p.head_tiles;
  const int head = kv_head * p.group + (hh - kv_head * p.head_tiles) * 16 + col - within * p.group;
  if (head >= (kv_head + 1) * p.group || t + within >= min(a.start[seq + 1], a.tokens)) return;
  const int2 item = p.items[((size_t)t * a.kv_heads) * p.head_tiles + hh];
  if (item.y <= 1 || item.x < 0 || item.x >= p.splits || item.y > p.splits - item.x) return;
  const float2* stats = p.stats + (size_t)item.x * p.rows + col;
  float m = -INFINITY;
  for (int i = tid; i < item.y; i += J) m = fmaxf(m, stats[(size_t)i * p.rows].x);
  for (int i = 1; i < 64; i *= 2) m = fmaxf(m, __shfl_xor(m, i));
  if ((tid & 63) == 0) part[tid >> 6] = m;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < J / 64; ++i) m = fmaxf(m, part[i]);
  const float ref = m == -INFINITY ? 0.0f : m;
  const int at = tid % (D / 4), lane = tid / (D / 4);
  const float* src = p.sums + ((size_t)item.x * p.rows + col) * D + at * 4;
  f32x4 o = {};
  float l = 0.0f;
  for (int i0 = 0; i0 < item.y; i0 += kJoinSplits) {
    const int n = min(kJoinSplits, item.y - i0);
    __syncthreads();
    for (int i = tid; i < n; i += J) {
      const float2 st = stats[(size_t)(i0 + i) * p.rows];
      const float w = __builtin_amdgcn_exp2f(st.x - ref);
      weight[i] = w;
      l = fmaf(w, st.y, l);
    }
    __syncthreads();
#pragma unroll 4
    for (int i = lane; i < n; i += kWide) o += weight[i] * *(const f32x4*)(src + (size_t)(i0 + i) * p.rows * D);
  }
  for (int i = 1; i < 64; i *= 2) l += __shfl_xor(l, i);
  __syncthreads();
  if ((tid & 63) == 0) part[tid >> 6] = l;
  sums[tid] = o;
  __syncthreads();
  if (tid >= D / 4) return;
  l = part[0];
#pragma unroll
  for (int i = 1; i < J / 64; ++i) l += part[i];
#pragma unroll
  for (int i = 1; i < kWide; ++i) o += sums[i * (D / 4) + tid];
  const float f = l == 0.0f ? 0.0f : 1.0f / l;
  ushort4 h;
  h.x = narrow<uint16_t>(o[0] * f), h.y = narrow<uint16_t>(o[1] * f);
  h.z = narrow<uint16_t>(o[2] * f), h.w = narrow<uint16_t>(o[3] * f);
  *(ushort4*)(g.y + ((size_t)(t + within) * g.heads + head) * D + tid * 4) = h;
}

// --- many new tokens ---------------------------------------------------------------

typedef float f32x16 __attribute__((ext_vector_type(16)));

// A tile of up to 128 rows (new tokens of a sequence x heads of a kv head) over
// all of its keys, 32 rows a wave.
//
// KT keys a step: a thread widens a quarter of a key's and of a value's row to
// f16 (their packed form was loaded a step before) and writes it to LDS, where
// the four waves read it: the conversion, not the bytes, would bound the
// kernel if each wave made its own.  S^T = K Q^T and O^T += V^T P^T on 32 x 32 x 16 matrix instructions:
// the first's result leaves a lane keys of one row that are the second's B
// operand as they stand, if V^T takes the keys in that order, which
// transposing reads of LDS give it.  Two workgroups fit a CU up to d = 128, so
// that one's exponentials run beside the other's products.  4,096 causal tokens
// of 32 heads over 8 kv heads, d = 128: 193 us, 710 TFLOP/s (466 us as a wave
// for each 16 rows); the exponentials and conversions take as long as the
// products there.
template <int D>
__global__ __launch_bounds__(256, D == 256 ? 1 : 2) void attention_tile_kernel(KvArgs a, AttnArgs g, int tile_tokens, int tiles_most) {
  constexpr int KT = D == 256 ? 32 : 64;
  constexpr int kKeyRow = D * 2 + 16, kValueRow = D * 2 + 32;  // bytes: no bank twice for the lanes of a read
  constexpr int kBuffer = KT * (kKeyRow + kValueRow);
  extern __shared__ __align__(16) uint8_t lds[];
  __shared__ uint32_t nan_lds[2][KT];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int row = lane & 31, half = lane >> 5;
  const int group = g.heads / a.kv_heads, kv_head = blockIdx.x % a.kv_heads;
  // the tiles with the most keys, a sequence's last, go first
  int tile = tiles_most - 1 - blockIdx.x / a.kv_heads;
  int seq = -1, start = 0, count = 0;
  for (int b0 = 0, before = 0; b0 < a.batch; b0 += 64) {
    const int b = b0 + lane;
    int t0 = 0, n = 0;
    if (b < a.batch) {
      t0 = max(a.start[b], 0);
      n = max(min(a.start[b + 1], a.tokens) - t0, 0);
    }
    const int tiles = (n + tile_tokens - 1) / tile_tokens;
    int upto = tiles;
    for (int i = 1; i < 64; i *= 2) {
      const int v = __shfl_up(upto, i);
      if (lane >= i) upto += v;
    }
    const unsigned long long hit = __ballot(tile >= before + upto - tiles && tile < before + upto);
    if (hit) {
      const int src = __ffsll(hit) - 1;
      seq = b0 + src;
      tile = __builtin_amdgcn_readfirstlane(tile - before - __shfl(upto - tiles, src));
      start = __builtin_amdgcn_readfirstlane(__shfl(t0, src));
      count = __builtin_amdgcn_readfirstlane(__shfl(n, src));
      break;
    }
    before += __shfl(upto, 63);
  }
  if (seq < 0) return;
  const long long table_keys = (long long)a.max_pages << a.page_shift;
  const long long raw = a.len[seq], len = min(max(raw, 0ll), table_keys);
  const int skip = tile * tile_tokens, mine = min(count - skip, tile_tokens);
  const long long pos0 = raw - count + skip, pos1 = pos0 + mine - 1;
  // this lane's row
  const int r = wave * 32 + row, within = r / group, head = kv_head * group + r - within * group;
  const bool real = within < mine;
  const int token = start + skip + within;
  const long long pos = pos0 + within;
  const int hi = !real ? 0 : (int)(g.causal ? max(0ll, min(len, pos + 1)) : len);
  const int lo = !real || g.window <= 0 ? 0 : (int)max(0ll, pos - g.window + 1);
  const int most = (int)(g.causal ? max(0ll, min(len, pos1 + 1)) : len);  // keys that some row sees: [from, most)
  const int from = g.window > 0 ? (int)min((long long)most, max(0ll, pos0 - g.window + 1)) : 0;
  const int every = (int)(g.causal ? max(0ll, min(len, pos0 + 1)) : len);  // that all rows see, up to here
  const int all_from = g.window > 0 ? (int)max(0ll, pos1 - g.window + 1) : 0;
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
  float m = -INFINITY, l = 0.0f;
  uint32_t nan_blocks = 0;
  const int j0 = from & ~15, steps = (most - j0 + KT - 1) / KT;
  const int32_t* table = a.table + (size_t)seq * a.max_pages;
  const int mask = (1 << a.page_shift) - 1;
  // the page of key `lane` of a step, or -1
  auto page_of = [&](int step) {
    const long long j = (long long)j0 + (long long)step * KT + lane;
    const int page = lane < KT && j < most ? table[j >> a.page_shift] : -1;
    return page < a.num_pages ? page : -1;
  };
  // this thread's part of the widening: a quarter of one key's row
  const bool does_k = KT == 64 || wave < 2, does_v = KT == 64 || wave >= 2;
  const int key = (tid >> 2) % KT, quarter = tid & 3;
  Piece<D> k, v;
  auto fetch = [&](int step, int pages) {
    const int j = j0 + step * KT + key;
    const int page = max(__shfl(pages, key), 0);  // a key on no page is seen by no row: any row's bytes will do
    const size_t at = (((size_t)page * a.kv_heads + kv_head) << a.page_shift) + (j & mask);
    if (does_k) k.load(a.kc, a.ks, at, quarter);
    if (does_v) v.load(a.vc, a.vs, at, quarter);
  };
  auto whole = [&](int step, unsigned long long there) {
    const int j = j0 + step * KT;
    return there == ~0ull >> (64 - KT) && j + KT <= every && j >= all_from;
  };
  auto widen_to = [&](int step, unsigned long long there) {
    uint8_t* kb = lds + (step & 1) * kBuffer + key * kKeyRow + quarter * (D / 2);
    uint8_t* vb = lds + (step & 1) * kBuffer + KT * kKeyRow + key * kValueRow + quarter * (D / 2);
    if (does_k) {
#pragma unroll
      for (int i = 0; i < D / 32; ++i) *(f16x8*)(kb + i * 16) = k.eight(i);
    }
    if (does_v) {
      if (!whole(step, there)) {
        // values that no row sees must not reach the sums, whatever they hold,
        // nor those that only some see, if they are NaN
        const int j = j0 + step * KT + key;
        if (!(there >> key & 1) || j >= most || j < from) v.clear();
        const uint32_t own = v.nan_bits(quarter);
        uint32_t bits = own | __shfl_xor(own, 1);
        bits |= __shfl_xor(bits, 2);
        if (own) v.clear_nan();
        if (quarter == 0) nan_lds[step & 1][key] = bits;
      }
#pragma unroll
      for (int i = 0; i < D / 32; ++i) *(f16x8*)(vb + i * 16) = v.eight(i);
    }
  };
  unsigned long long there = 0, there_next = 0;
  if (steps > 0) {
    int pages = page_of(0);
    there = __ballot(pages >= 0);
    fetch(0, pages);
    widen_to(0, there);
    if (steps > 1) {
      pages = page_of(1);
      there_next = __ballot(pages >= 0);
      fetch(1, pages);
    }
  }
  int pages = steps > 2 ? page_of(2) : -1;
  __syncthreads();
  for (int step = 0; step < steps; ++step) {
    unsigned long long there_after = 0;
    if (step + 1 < steps) {
      widen_to(step + 1, there_next);
      if (step + 2 < steps) {
        there_after = __ballot(pages >= 0);
        fetch(step + 2, pages);
        if (step + 3 < steps) pages = page_of(step + 3);
      }
    }
    const uint8_t* kb = lds + (step & 1) * kBuffer;
    const uint8_t* vb = kb + KT * kKeyRow;
    f32x16 t[KT / 32];
#pragma unroll
    for (int u = 0; u < KT / 32; ++u) {
      t[u] = f32x16{};
#pragma unroll
      for (int i = 0; i < D / 16; ++i) {
        const f16x8 x = *(const f16x8*)(kb + (u * 32 + row) * kKeyRow + i * 32 + half * 16);
        t[u] = __builtin_amdgcn_mfma_f32_32x32x16_f16(x, q[i], t[u], 0, 0, 0);
      }
    }
    uint32_t see = ~0u;
    if (!whole(step, there)) {
      see = 0;
#pragma unroll
      for (int u = 0; u < KT / 32; ++u)
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const int c = u * 32 + 8 * (e / 4) + 4 * half + e % 4, j = j0 + step * KT + c;
          const bool yes = (there >> c & 1) && j < hi && j >= lo;
          see |= (uint32_t)yes << (u * 16 + e);
          t[u][e] = yes ? t[u][e] : -INFINITY;
        }
      const uint32_t any = lane < KT ? nan_lds[step & 1][lane] : 0u;
      if (__ballot(any != 0)) {
#pragma unroll
        for (int u = 0; u < KT / 32; ++u)
#pragma unroll
          for (int e = 0; e < 16; ++e)
            if (see >> (u * 16 + e) & 1) nan_blocks |= nan_lds[step & 1][u * 32 + 8 * (e / 4) + 4 * half + e % 4];
      }
    }
    float top = t[0][0];
#pragma unroll
    for (int u = 0; u < KT / 32; ++u)
#pragma unroll
      for (int e = 0; e < 16; ++e) top = fmaxf(top, t[u][e]);
    if (__ballot(m == -INFINITY ? top > m : (top - m) * g.scale > 8.0f)) {
      const float now = fmaxf(m, fmaxf(top, __shfl_xor(top, 32)));
      const float f = now == m ? 1.0f : m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f((m - now) * g.scale);
      l *= f;
#pragma unroll
      for (int i = 0; i < D / 32; ++i) o[i] *= f;
      m = now;
    }
    // 2^6 times: a p of 2^-20 of the largest is still a normal f16 number
    const float ref = (m == -INFINITY ? 0.0f : m * g.scale) - 6.0f;
    f16x8 p[KT / 16];
#pragma unroll
    for (int u = 0; u < KT / 32; ++u)
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        float x = __builtin_amdgcn_exp2f(fmaf(t[u][e], g.scale, -ref));
        x = see >> (u * 16 + e) & 1 ? x : 0.0f;
        l += x;
        p[u * 2 + e / 8][e % 8] = (_Float16)x;
      }
#pragma unroll
    for (int i = 0; i < D / 32; ++i)
#pragma unroll
      for (int u = 0; u < KT / 16; ++u) {
        // four groups of 16 lanes: 4 keys x 16 elements each
        typedef __attribute__((address_space(3))) s16x4* Lds;
        typedef short s16x8 __attribute__((ext_vector_type(8)));
        const int e = lane & 15;
        const uint8_t* src = vb + (u * 16 + 4 * half + (e >> 2)) * kValueRow + i * 64 + ((lane >> 4) & 1) * 32 + (e & 3) * 8;
        const s16x4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((Lds)src);
        const s16x4 y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((Lds)(src + 8 * kValueRow));
        const s16x8 xy = {x[0], x[1], x[2], x[3], y[0], y[1], y[2], y[3]};
        o[i] = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, xy), p[u], o[i], 0, 0, 0);
      }
    there = there_next;
    there_next = there_after;
    __syncthreads();
  }
  l += __shfl_xor(l, 32);
  nan_blocks |= __shfl_xor(nan_blocks, 32);
  if (!real) return;
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
void launch_tiles(hipStream_t st, const KvArgs& a, const AttnArgs& g) {
  constexpr int kKeys = D == 256 ? 32 : 64, kLds = 2 * kKeys * (D * 4 + 48);
  const int tile_tokens = 128 / (g.heads / a.kv_heads), tiles = std::min(a.tokens, a.tokens / tile_tokens + a.batch);
  hipLaunchKernelGGL(attention_tile_kernel<D>, dim3((unsigned)(tiles * a.kv_heads)), dim3(256), kLds, st, a, g,
                     tile_tokens, tiles);
}

template <int D>
void launch_splits(hipStream_t st, const KvArgs& a, const AttnArgs& g, const SplitArgs& p) {
  // Rows of few splits are many: a wave each then.
  const dim3 rows((unsigned)a.tokens, (unsigned)(a.kv_heads * p.head_tiles), (unsigned)p.rows);
  const bool few = (long long)a.tokens * g.heads <= 512;
  hipLaunchKernelGGL(attention_split_kernel<D>, dim3((unsigned)p.splits), dim3(64), 0, st, a, g, p);
  if (!p.join) return;  // a split takes all keys that the table has room for
  if (few)
    hipLaunchKernelGGL((attention_join_kernel<D, 512>), rows, dim3(512), 0, st, a, g, p);
  else
    hipLaunchKernelGGL((attention_join_kernel<D, 64>), rows, dim3(64), 0, st, a, g, p);
}

}  // namespace

size_t attention_space(const KvArgs& a, const AttnArgs& g, SplitArgs* p) {
  p->group = g.heads / a.kv_heads;
  // Whole tiles are faster where there are enough of them, and full: 512 new
  // tokens of 32 heads 24 us, 53 us split; 256 of them after 8,192 keys (64
  // tiles, 8,192 rows) 250 us, 110 us split; 8 sequences of up to 64 after
  // 2,048 keys 68 us, 31 us split.
  p->whole = p->group <= 128 && (long long)a.tokens * g.heads >= 12288 &&
             (long long)a.tokens * p->group >= 128ll * a.batch;
  if (p->whole) return 0;
  p->head_tiles = (p->group + 15) / 16;
  p->tile_tokens = std::max(1, 16 / p->group);
  const long long tiles = std::min<long long>(a.tokens, a.tokens / p->tile_tokens + (long long)a.batch);
  const long long heads = (long long)a.kv_heads * p->head_tiles;
  p->waves = 2048;
  p->waves = a.d == 256 ? 1024 : 2048;  // that the chip holds at a time
  // A split takes two steps of 64 keys or more, or all of them where joining
  // would take longer: one sequence of 1,024 keys 12.2 us in splits of two, 20.9
  // us in splits of eight; 64 of up to 512 17.5 us split, 14.1 us whole.
  const int steps = ((a.max_pages << a.page_shift) + kChunk - 1) / kChunk;  // of the longest sequence
  p->join = steps > (tiles * heads >= 256 ? 8 : 4);
  p->least = p->join ? 2 : 8;
  p->splits = (int)(tiles * heads + p->waves + 1);
  p->rows = std::min(16, p->group * p->tile_tokens);
  p->stats_at = (size_t)p->splits * p->rows * a.d * 4;
  p->items_at = p->stats_at + (size_t)p->splits * p->rows * 8;
  return p->items_at + (size_t)a.tokens * heads * 8;
}

void launch_attention(hipStream_t st, const KvArgs& a, const AttnArgs& g, SplitArgs p, void* space) {
  auto run = [&](auto d) {
    constexpr int D = decltype(d)::value;
    p.whole ? launch_tiles<D>(st, a, g) : launch_splits<D>(st, a, g, p);
  };
  if (!p.whole) {
    p.sums = (float*)space;
    p.stats = (float2*)((char*)space + p.stats_at);
    p.items = (int2*)((char*)space + p.items_at);
  }
  if (a.d == 64)
    run(std::integral_constant<int, 64>{});
  else if (a.d == 128)
    run(std::integral_constant<int, 128>{});
  else
    run(std::integral_constant<int, 256>{});
  DW_HIP(hipGetLastError());
}

}  // namespace dw
