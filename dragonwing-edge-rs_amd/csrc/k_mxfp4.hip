// Rows to MXFP4 and back (mxfp4.h).
//
// Both are bound by memory: x is read once, q and the scales are written once
// (or the reverse).  A thread takes 8 elements, so that a wave reads 1 or 2
// KiB in one piece and writes 256 bytes of q; the four threads of a block
// share its largest magnitude by two lane permutes.  Rows whose length is a
// multiple of 32 have no ends inside: they are taken as one row.
//
// 8,191 x 4,099 f32: quantized in 33 us (4.6 TB/s, a large copy reaches 4.8),
// read back as f32 in 38 us (4.0 TB/s).
#include <algorithm>

#include "dw_common.h"
#include "mxfp4.h"

namespace dw {

namespace {

// blockDim = (threads along a row, rows)
template <typename T>
__global__ __launch_bounds__(256) void quantize_mxfp4_kernel(const T* __restrict__ x, uint32_t* __restrict__ q,
                                                             uint8_t* __restrict__ scales, size_t rows, size_t k) {
  const size_t units = (k + 31) / 32 * 4;
  const size_t u = (size_t)blockIdx.x * blockDim.x + threadIdx.x;
  if (u >= units) return;  // whole blocks of 32 elements: no part of a quad
  for (size_t r = (size_t)blockIdx.y * blockDim.y + threadIdx.y; r < rows; r += (size_t)gridDim.y * blockDim.y) {
    const T* p = x + r * k + u * 8;
    float v[8];
    if (u * 8 + 8 <= k) {
      const Loose<T, 8> l = load_loose<T, 8>(p);
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = widen(l.v[i]);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = u * 8 + i < k ? widen(p[i]) : 0.0f;
    }
    uint32_t big = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) big = max(big, __builtin_bit_cast(uint32_t, v[i]) & 0x7FFFFFFFu);
    const uint32_t b = mx_scale_byte(max_of_quad(big), 0);
    q[r * units + u] = b == 255u ? 0u : mx_encode8(v, mx_scale(b));
    if ((u & 3) == 0) scales[r * (units / 4) + u / 4] = (uint8_t)b;
  }
}

// E elements a thread: 16 bytes of y, so that a wave's stores are one piece.
template <typename T, int E>
__global__ __launch_bounds__(256) void dequantize_mxfp4_kernel(const uint8_t* __restrict__ q,
                                                               const uint8_t* __restrict__ scales,
                                                               T* __restrict__ y, size_t rows, size_t k) {
  const size_t blocks = (k + 31) / 32;
  const size_t u = (size_t)blockIdx.x * blockDim.x + threadIdx.x;
  if (u * E >= k) return;
  for (size_t r = (size_t)blockIdx.y * blockDim.y + threadIdx.y; r < rows; r += (size_t)gridDim.y * blockDim.y) {
    const uint8_t* at = q + r * blocks * 16 + u * (E / 2);
    float v[8];
    mx_decode8(E == 8 ? *(const uint32_t*)at : *(const uint16_t*)at, mx_scale(scales[r * blocks + u / (32 / E)]), v);
    T* p = y + r * k + u * E;
    Loose<T, E> l;
#pragma unroll
    for (int i = 0; i < E; ++i) l.v[i] = narrow<T>(v[i]);
    if (u * E + E <= k) {
      store_loose<T, E>(p, l);
    } else {
#pragma unroll
      for (int i = 0; i < E; ++i)
        if (u * E + i < k) p[i] = l.v[i];
    }
  }
}

struct Shape {
  size_t rows, k;
  dim3 grid, block;
};
Shape shape_of(size_t rows, size_t k, int each) {  // each: elements of a thread
  Shape s{rows, k, {}, {}};
  if (k % 32 == 0 && rows * k <= (size_t)1 << 33) {  // a grid has under 2^32 threads
    s.k = rows * k;
    s.rows = 1;
  }
  const size_t units = (s.k + 31) / 32 * (32 / each);
  unsigned tx = 4;
  while (tx < 256 && tx < units) tx *= 2;
  const unsigned ty = 256 / tx;
  s.block = dim3(tx, ty);
  s.grid = dim3((unsigned)((units + tx - 1) / tx), (unsigned)std::min<size_t>((s.rows + ty - 1) / ty, 65535));
  return s;
}

}  // namespace

void launch_quantize_mxfp4(hipStream_t st, int dtype, const void* x, void* q, void* scales, size_t rows, size_t k) {
  const Shape s = shape_of(rows, k, 8);
  if (dtype == F16)
    hipLaunchKernelGGL(quantize_mxfp4_kernel<uint16_t>, s.grid, s.block, 0, st, (const uint16_t*)x, (uint32_t*)q,
                       (uint8_t*)scales, s.rows, s.k);
  else
    hipLaunchKernelGGL(quantize_mxfp4_kernel<float>, s.grid, s.block, 0, st, (const float*)x, (uint32_t*)q,
                       (uint8_t*)scales, s.rows, s.k);
  DW_HIP(hipGetLastError());
}

void launch_dequantize_mxfp4(hipStream_t st, int dtype, const void* q, const void* scales, void* y, size_t rows,
                             size_t k) {
  const Shape s = shape_of(rows, k, dtype == F16 ? 8 : 4);
  if (dtype == F16)
    hipLaunchKernelGGL((dequantize_mxfp4_kernel<uint16_t, 8>), s.grid, s.block, 0, st, (const uint8_t*)q,
                       (const uint8_t*)scales, (uint16_t*)y, s.rows, s.k);
  else
    hipLaunchKernelGGL((dequantize_mxfp4_kernel<float, 4>), s.grid, s.block, 0, st, (const uint8_t*)q,
                       (const uint8_t*)scales, (float*)y, s.rows, s.k);
  DW_HIP(hipGetLastError());
}

}  // namespace dw
