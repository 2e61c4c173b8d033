// Attention over a cache of keys and values in MXFP4 pages, and what writes
// the cache.
//
// A page holds page_size rows of each kv head, [page][head][slot][d / 2]
// bytes and [page][head][slot][d / 32] scales: the rows are MXFP4 rows of d
// elements (mxfp4.h), so the cache's values can be read back as such rows.
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

// The plain kernel: a wave for each new token and head, 64 keys a step.
__global__ __launch_bounds__(64) void attention_plain_kernel(KvArgs a, AttnArgs g) {
  __shared__ int found;
  __shared__ float qs[256], ps[64];
  __shared__ size_t rows[64];
  const int t = blockIdx.x, h = blockIdx.y, lane = threadIdx.x, kh = h / (g.heads / a.kv_heads);
  const int seq = sequence_of(a.start, a.batch, t, &found);
  if (seq >= a.batch || t < a.start[seq]) return;
  for (int d = lane; d < a.d; d += 64) qs[d] = h2f_ieee(g.q[(size_t)t * g.q_stride + g.q_off + (size_t)h * a.d + d]);
  __syncthreads();
  const long long most = (long long)a.max_pages << a.page_shift;
  const long long len = a.len[seq] < 0 ? 0 : min((long long)a.len[seq], most);
  const long long pos = (long long)a.len[seq] - a.start[seq + 1] + t;
  const long long end = g.causal ? min(len, pos + 1) : len;
  const long long begin = g.window > 0 ? max(0ll, pos - g.window + 1) : 0;
  float m = -INFINITY, l = 0.0f, o[4] = {};
  for (long long j0 = begin; j0 < end; j0 += 64) {
    const long long j = j0 + lane;
    float s = -INFINITY;
    size_t row = ~(size_t)0;
    if (j < end) {
      const int page = a.table[(size_t)seq * a.max_pages + (j >> a.page_shift)];
      if (page >= 0 && page < a.num_pages) {
        row = (((size_t)page * a.kv_heads + kh) << a.page_shift) + (j & ((1 << a.page_shift) - 1));
        s = 0.0f;
        for (int u = 0; u < a.d / 8; ++u) {
          float v[8];
          mx_decode8(a.kc[row * (a.d / 8) + u], mx_scale(a.ks[row * (a.d / 32) + u / 4]), v);
          for (int e = 0; e < 8; ++e) s = fmaf(qs[u * 8 + e], v[e], s);
        }
        s *= g.scale;
      }
    }
    float mx = s;
    for (int i = 1; i < 64; i *= 2) mx = fmaxf(mx, __shfl_xor(mx, i));
    const float now = fmaxf(m, mx);
    const float ref = now == -INFINITY ? 0.0f : now;
    const float p = row == ~(size_t)0 ? 0.0f : expf(s - ref);
    float sum = p;
    for (int i = 1; i < 64; i *= 2) sum += __shfl_xor(sum, i);
    const float f = expf(m - ref);
    l = l * f + sum;
    m = now;
    ps[lane] = p;
    rows[lane] = row;
    __syncthreads();
    for (int i = 0; i < 4; ++i) o[i] *= f;
    for (int e = 0; e < 64; ++e) {
      if (rows[e] == ~(size_t)0) continue;
      for (int i = 0; i * 64 + lane < a.d; ++i) {
        const int d = i * 64 + lane;
        float v[8];
        mx_decode8(a.vc[rows[e] * (a.d / 8) + d / 8], mx_scale(a.vs[rows[e] * (a.d / 32) + d / 32]), v);
        float x = v[0];
        for (int b = 1; b < 8; ++b) x = (d & 7) == b ? v[b] : x;
        o[i] = fmaf(ps[e], x, o[i]);
      }
    }
    __syncthreads();
  }
  for (int i = 0; i * 64 + lane < a.d; ++i)
    g.y[((size_t)t * g.heads + h) * a.d + i * 64 + lane] = narrow<uint16_t>(l == 0.0f ? 0.0f : o[i] / l);
}

}  // namespace

void launch_kv_append(hipStream_t st, const KvArgs& a, const void* k, size_t k_stride, size_t k_off, const void* v,
                      size_t v_stride, size_t v_off) {
  hipLaunchKernelGGL(kv_append_kernel, dim3((unsigned)a.tokens), dim3(256), 0, st, a, (const uint16_t*)k, k_stride,
                     k_off, (const uint16_t*)v, v_stride, v_off);
  DW_HIP(hipGetLastError());
}

void launch_attention(hipStream_t st, const KvArgs& a, const AttnArgs& g) {
  hipLaunchKernelGGL(attention_plain_kernel, dim3((unsigned)a.tokens, (unsigned)g.heads), dim3(64), 0, st, a, g);
  DW_HIP(hipGetLastError());
}

}  // namespace dw
