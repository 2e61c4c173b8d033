// Products of rows (f16 or MXFP4) and MXFP4 weights: C = act(A W^T + bias).
#include <algorithm>

#include "dw_common.h"
#include "mxfp4.h"

namespace dw {

namespace {

// bias, activation and the one rounding of a sum
template <bool H>
__device__ __forceinline__ void finish(const GemmMxArgs& a, size_t row, size_t col, float s) {
  if (a.bias) s += H ? h2f_ieee(((const uint16_t*)a.bias)[col]) : ((const float*)a.bias)[col];
  if (a.act == ACT_RELU) s = s < 0.0f ? 0.0f : s;  // a NaN stays
  if (a.act == ACT_SILU) s = s / (1.0f + expf(-s));
  if (H)
    ((uint16_t*)a.c)[row * a.n + col] = narrow<uint16_t>(s);
  else
    ((float*)a.c)[row * a.n + col] = s;
}

template <bool MX, bool H>
__global__ __launch_bounds__(256) void gemm_mx_plain_kernel(GemmMxArgs a) {
  const size_t blocks = (a.k + 31) / 32, total = (size_t)a.m * a.n;
  for (size_t i = (size_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (size_t)gridDim.x * 256) {
    const size_t row = i / a.n, col = i - row * a.n;
    const uint32_t* w = (const uint32_t*)a.w + col * blocks * 4;
    float sum = 0.0f;
    for (size_t b = 0; b < blocks; ++b) {
      const float sw = mx_scale(a.ws[col * blocks + b]);
      for (int j = 0; j < 4; ++j) {
        float v[8], u[8];
        mx_decode8(w[b * 4 + j], sw, v);
        if (MX) mx_decode8(((const uint32_t*)a.a)[(row * blocks + b) * 4 + j], mx_scale(a.as[row * blocks + b]), u);
        for (int e = 0; e < 8; ++e) {
          const size_t at = b * 32 + j * 8 + e;
          if (at < (size_t)a.k) sum = fmaf(MX ? u[e] : h2f_ieee(((const uint16_t*)a.a)[row * a.k + at]), v[e], sum);
        }
      }
    }
    finish<H>(a, row, col, sum);
  }
}

}  // namespace

void launch_gemm_mx(hipStream_t st, const GemmMxArgs& a) {
  const size_t total = (size_t)a.m * a.n;
  const dim3 grid((unsigned)std::min<size_t>((total + 255) / 256, 1u << 20));
  auto* k = a.as ? (a.c_half ? gemm_mx_plain_kernel<true, true> : gemm_mx_plain_kernel<true, false>)
                 : (a.c_half ? gemm_mx_plain_kernel<false, true> : gemm_mx_plain_kernel<false, false>);
  hipLaunchKernelGGL(k, grid, dim3(256), 0, st, a);
  DW_HIP(hipGetLastError());
}

}  // namespace dw
