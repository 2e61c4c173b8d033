// Rotary positions over several axes.
//
// Pair i of a head turns by the angle pos[axis(i)][token] * freq(i).  The
// angle is formed in turns and in 64 bits, where a position of millions still
// leaves 2^-30 of a turn, and only its fraction becomes f32: in f32 the
// angle of position 500,000 would be off by 0.03 radians.  The cosines and
// sines of a token are computed once and shared by its heads through LDS.
// Bound by memory: every element is read and written once.  12,289 tokens x 24
// heads x 80 f32: 40 us (4.8 TB/s, what a large copy reaches).
#include <algorithm>

#include "dw_common.h"
#include "mxfp4.h"

namespace dw {

namespace {

constexpr int kMaxHalf = 128;  // pairs of a head

// ADJ: a pair is two adjacent elements, else elements i and i + rotary / 2.
// V: pairs of a thread's step (rotary / 2 is a multiple of V).  A thread's
// first elements are loaded before the cosines are computed.
template <typename T, bool ADJ, int V>
__global__ __launch_bounds__(256) void rope_kernel(RopeArgs a) {
  __shared__ float2 turn[kMaxHalf];
  const size_t t = blockIdx.x;
  const T* x = (const T*)a.x + t * a.x_stride + a.x_off;
  T* y = (T*)a.y + t * a.y_stride + a.y_off;
  const int steps = a.half / V;                           // of a head's pairs
  const int rest = a.copy ? a.head_dim - 2 * a.half : 0;  // elements that do not turn
  const int each = steps + (rest + 2 * V - 1) / (2 * V), total = a.heads * each;
  Loose<T, V> p = {}, q = {};
  int i = 0;               // first pair, or first element behind the pairs
  size_t at0 = 0, at1 = 0;
  bool pairs = false;
  auto load = [&](int u) {
    const int h = u / each, j = u - h * each;
    const size_t base = (size_t)h * a.head_dim;
    pairs = j < steps;
    if (pairs) {
      i = j * V;
      at0 = base + (ADJ ? 2 * i : i), at1 = ADJ ? at0 + V : at0 + a.half;
    } else {
      i = (j - steps) * 2 * V;
      at0 = base + 2 * a.half + i, at1 = at0 + V;
      if (i + 2 * V > rest) return;  // the last few come one by one
    }
    p = load_loose<T, V>(x + at0), q = load_loose<T, V>(x + at1);
  };
  int u = blockIdx.y * 256 + threadIdx.x;
  if (u < total) load(u);
  if ((int)threadIdx.x < a.half) {
    const int32_t pos = a.pos[(size_t)a.table.axis[threadIdx.x] * a.tokens + t];
    const double w = (double)pos * a.table.freq[threadIdx.x];
    const float f = (float)(w - rint(w));  // in [-1/2, 1/2] turns
    float s, c;
    sincospif(2.0f * f, &s, &c);
    turn[threadIdx.x] = make_float2(c, s);
  }
  __syncthreads();
  while (u < total) {
    if (pairs) {
      float lo[V], hi[V];  // first and second elements of the pairs
#pragma unroll
      for (int e = 0; e < V; ++e) {
        lo[e] = widen(ADJ ? (2 * e < V ? p.v[2 * e % V] : q.v[2 * e % V]) : p.v[e]);
        hi[e] = widen(ADJ ? (2 * e + 1 < V ? p.v[(2 * e + 1) % V] : q.v[(2 * e + 1) % V]) : q.v[e]);
      }
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const float2 cs = turn[i + e];
        const float r0 = fmaf(-hi[e], cs.y, lo[e] * cs.x), r1 = fmaf(lo[e], cs.y, hi[e] * cs.x);
        if (ADJ) {
          (2 * e < V ? p.v[2 * e % V] : q.v[2 * e % V]) = narrow<T>(r0);
          (2 * e + 1 < V ? p.v[(2 * e + 1) % V] : q.v[(2 * e + 1) % V]) = narrow<T>(r1);
        } else {
          p.v[e] = narrow<T>(r0);
          q.v[e] = narrow<T>(r1);
        }
      }
    }
    if (pairs || i + 2 * V <= rest) {
      store_loose<T, V>(y + at0, p);
      store_loose<T, V>(y + at1, q);
    } else {
      for (int e = 0; i + e < rest; ++e) y[at0 + e] = x[at0 + e];
    }
    u += gridDim.y * 256;
    if (u < total) load(u);
  }
}

template <typename T, bool ADJ>
void launch(hipStream_t st, const RopeArgs& a, dim3 grid) {
  auto* k = a.half % 8 == 0 && sizeof(T) == 2 ? rope_kernel<T, ADJ, 8>
            : a.half % 4 == 0                 ? rope_kernel<T, ADJ, 4>
                                              : rope_kernel<T, ADJ, 1>;
  hipLaunchKernelGGL(k, grid, dim3(256), 0, st, a);
}

}  // namespace

void launch_rope(hipStream_t st, int dtype, const RopeArgs& a, int adjacent) {
  // few tokens: their heads over several workgroups
  const dim3 grid((unsigned)a.tokens, a.tokens < 256 ? (unsigned)std::min(8, (a.heads * a.head_dim + 4095) / 4096) : 1u);
  if (dtype == F16)
    adjacent ? launch<uint16_t, true>(st, a, grid) : launch<uint16_t, false>(st, a, grid);
  else
    adjacent ? launch<float, true>(st, a, grid) : launch<float, false>(st, a, grid);
  DW_HIP(hipGetLastError());
}

}  // namespace dw
