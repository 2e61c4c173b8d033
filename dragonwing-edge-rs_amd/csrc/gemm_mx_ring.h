// Tiles of 256 x 256 of the products with MXFP4 weights whose two halves take turns
// at LDS and at the matrix cores (gemm_mx.h has the smaller ones).
#pragma once

#include "gemm_mx.h"

namespace dw {

namespace {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

// Eight waves, two along the rows of A and four along those of W, 8 x 4 tiles of 16 x
// 16 each.  LDS holds kRing stages of K: three of 64 elements of f16 rows, two of 256 of
// MXFP4 ones, whole lines of A of 128 bytes and, where there is room, of W.
//
// A stage comes in two parts of one matrix instruction's depth, and a part in two
// phases with a meeting of all waves behind each: reads of LDS with the conversions,
// then products.  Waves 4 to 7, which share their SIMDs with waves 0 to 3, are a phase
// behind, so that a SIMD's matrix core has one wave's products while the other
// reads.  Loads of the stage that takes the place of the last one go out with a stage's first
// reads; the wait before a stage leaves those behind it in flight.
//
// Reads of LDS are written out, each block with its wait: the compiler, which does
// not know which loads write which place, would wait for all of them, and it waits for
// all of them, too, for a load to a register; so scales come to LDS by themselves, 16 bytes a
// row and 512 elements.
//
// 8,192 x 14,336 x 4,096 for two experts, f16 rows: 762 us (1.26 PFLOP/s, 1.48 along K
// alone; a library's f16 product reaches 1.58), 775 us with all waves in step, 930 us
// with odd waves behind, 810 us in the tiles of gemm_mx.h.  65,536 x 4,096 x 4,096 for eight
// experts, MXFP4 rows: 683 us (3.2 PFLOP/s, 4.7 along K alone), 693 us in step, 722 us
// with odd waves behind, 732 us in stages of 128 elements, half a line, and 714 us in the others' tiles.
// What is left is a tile's ends: 4 us until its first products and 7 to 9 us of stores.
template <bool MX>
struct Ring {
  static constexpr int kRing = MX ? 2 : 3, kDepth = MX ? 256 : 64;
  static constexpr int TM = 8, TN = 4, kRowsA = 256, kRowsW = 256;
  static constexpr int kLineA = 128, kLineW = MX ? 128 : 32;  // bytes of a row and stage
  static constexpr int kA = kRowsA * kLineA, kW = kRowsW * kLineW, kStage = kA + kW;
  static constexpr int kSpan = 512 / kDepth;  // stages of a scale row's 16 bytes
  static constexpr int kScaleRows = (MX ? kRowsA : 0) + kRowsW, kScales = kScaleRows * 16;
  static constexpr int kLds = kRing * kStage + 2 * kScales;
  static constexpr int kLoadsA = kA / 8192, kLoadsW = kW / 8192, kLoads = kLoadsA + kLoadsW;  // a wave's, of 1 KiB

  const GemmMxArgs& g;
  uint8_t* lds;
  int m0, n0, wave, lane, col, quad, wm, wn, blocks;
  uint32_t at_a[kLoadsA], at_w[kLoadsW];  // a lane's pieces of the first stage: in 16 bytes from A's row 0, from the tile's rows of W
  const uint8_t *base_w, *scales;         // scales: of this lane's row

  __device__ __forceinline__ Ring(const GemmMxArgs& args, uint8_t* shared, int row0, int col0, const RowList& list)
      : g(args), lds(shared), m0(row0), n0(col0) {
    wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    lane = threadIdx.x & 63, col = lane & 15, quad = lane >> 4, wm = wave & 1, wn = wave >> 1;
    blocks = (g.k + 31) / 32;
    const uint32_t row_a = MX ? blocks : g.lda / 8;  // in 16 bytes
    const size_t row_w = (size_t)blocks * 16;
    base_w = g.w + n0 * row_w;
#pragma unroll
    for (int i = 0; i < kLoadsA; ++i) {
      const int r = row_of_a(i), in = min(r, g.m - 1 - m0);  // rows behind the end are not stored
      at_a[i] = list.row(m0 + in) * row_a + piece_a(r);
    }
#pragma unroll
    for (int i = 0; i < kLoadsW; ++i) at_w[i] = (uint32_t)(min(row_of_w(i), g.n - 1 - n0) * row_w) + piece_w(i) * 16;
    const int r = scale_row();
    scales = MX && r < kRowsA ? g.as + (size_t)list.row(m0 + min(r, g.m - 1 - m0)) * g.pitch
                              : g.ws + (size_t)(n0 + min(r - (MX ? kRowsA : 0), g.n - 1 - n0)) * g.pitch;
  }
  // Rows of scales, A's before W's, 64 a wave; those of W alone two waves bring.
  __device__ __forceinline__ int scale_row() const { return wave * 64 % kScaleRows + lane; }
  // Load i of this wave brings 64 pieces of 16 bytes, a lane one, to places side by
  // side.  The pieces of row r stand at their index xor a part of r, so that eight rows'
  // reads of one piece meet all banks; rows of W of 32 bytes stand 32 together, piece by
  // piece.
  __device__ __forceinline__ int row_of_a(int i) const { return (wave * kLoadsA + i) * (1024 / kLineA) + lane / (kLineA / 16); }
  __device__ __forceinline__ int row_of_w(int i) const {
    return MX ? (wave * kLoadsW + i) * 8 + lane / 8 : (wave * kLoadsW + i) * 32 + lane % 32;
  }
  __device__ __forceinline__ int piece_a(int r) const { return lane % 8 ^ (r & 7); }
  __device__ __forceinline__ int piece_w(int i) const { return MX ? lane % 8 ^ (row_of_w(i) & 7) : lane / 32; }

  // LAST: some of the stage's pieces may lie behind the end of K.
  template <bool LAST>
  __device__ __forceinline__ void load(int place, int stage) const {
    uint8_t* slot = lds + place * kStage;
    const uint8_t* pa = (const uint8_t*)g.a + (size_t)stage * kLineA;
    const uint8_t* pw = base_w + (size_t)stage * kLineW;
    const int left_a = (MX ? blocks : g.lda / 8) - stage * (kLineA / 16), left_w = blocks - stage * (kLineW / 16);
#pragma unroll
    for (int i = 0; i < kLoadsA; ++i) {
      const uint8_t* p = pa + (size_t)at_a[i] * 16;
      if (LAST && piece_a(row_of_a(i)) >= left_a) p = (const uint8_t*)kZeros;
      __builtin_amdgcn_global_load_lds((const void*)p, (LdsPtr)(slot + (wave * kLoadsA + i) * 1024), 16, 0, 0);
    }
#pragma unroll
    for (int i = 0; i < kLoadsW; ++i) {
      const uint8_t* p = pw + at_w[i];
      if (LAST && piece_w(i) >= left_w) p = (const uint8_t*)kZeros;
      __builtin_amdgcn_global_load_lds((const void*)p, (LdsPtr)(slot + kA + (wave * kLoadsW + i) * 1024), 16, 0, 0);
    }
  }
  // The 16 scale bytes of 512 elements of each row; behind the end some that are not read.
  __device__ __forceinline__ void load_scales(int span) const {
    const uint8_t* p = scales + (span * 16 < blocks ? span * 16 : 0);
    uint8_t* to = lds + kRing * kStage + (span & 1) * kScales + wave * 64 % kScaleRows * 16;
    __builtin_amdgcn_global_load_lds((const void*)p, (LdsPtr)to, 16, 0, 0);
  }
  static __device__ __forceinline__ uint32_t address(const uint8_t* p) { return (uint32_t)(uintptr_t)(LdsPtr)p; }

  // All but the last MORE of this wave's loads are done.
  template <int MORE>
  static __device__ __forceinline__ void wait() {
    static_assert(MORE < 16, "vmcnt's lower bits");
    __builtin_amdgcn_s_waitcnt(MORE | 7 << 4 | 15 << 8);
    asm volatile("" ::: "memory");
  }
  static __device__ __forceinline__ void meet() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
  }

  template <bool EXACT>
  __device__ __forceinline__ void multiply(int place, int stage, uint32_t* far, f32x4 (&acc)[TN][TM]) const {
    const uint8_t* slot = lds + place * kStage;
    const uint8_t* sc = lds + kRing * kStage + (stage / kSpan & 1) * kScales;
    // All loads of the stage after this one are done, those behind them (and, of the
    // next span's scales, in flight for two turns) may not be.
    auto settle = [&] {
      if (stage % kSpan <= kRing - 3)
        wait<(kRing - 2) * kLoads + 1>();
      else
        wait<(kRing - 2) * kLoads>();
    };
    if constexpr (MX) {
#pragma unroll
      for (int part = 0; part < 2; ++part) {
        const int turn = ((quad ^ (col & 7)) ^ part * 4) * 16;
        const uint32_t pa = address(slot + (wm * 128 + col) * 128 + turn), pw = address(slot + kA + (wn * 64 + col) * 128 + turn);
        const uint8_t* scq = sc + stage % kSpan * 8 + part * 4 + quad;
        const uint32_t sa = address(scq + (wm * 128 + col) * 16), sw = address(scq + (kRowsA + wn * 64 + col) * 16);
        u32x4 x[TM], y[TN];
        uint32_t fx[TM], fw[TN];
        asm volatile(
            "ds_read_u8 %8, %26\n\tds_read_u8 %9, %26 offset:256\n\tds_read_u8 %10, %26 offset:512\n\t"
            "ds_read_u8 %11, %26 offset:768\n\tds_read_u8 %12, %26 offset:1024\n\tds_read_u8 %13, %26 offset:1280\n\t"
            "ds_read_u8 %14, %26 offset:1536\n\tds_read_u8 %15, %26 offset:1792\n\tds_read_u8 %20, %27\n\t"
            "ds_read_u8 %21, %27 offset:256\n\tds_read_u8 %22, %27 offset:512\n\tds_read_u8 %23, %27 offset:768\n\t"
            "ds_read_b128 %16, %25\n\tds_read_b128 %0, %24\n\tds_read_b128 %1, %24 offset:2048\n\tds_read_b128 %2, %24 offset:4096\n\t"
            "ds_read_b128 %3, %24 offset:6144\n\tds_read_b128 %4, %24 offset:8192\n\tds_read_b128 %5, %24 offset:10240\n\t"
            "ds_read_b128 %6, %24 offset:12288\n\tds_read_b128 %7, %24 offset:14336\n\tds_read_b128 %17, %25 offset:2048\n\t"
            "ds_read_b128 %18, %25 offset:4096\n\tds_read_b128 %19, %25 offset:6144\n\ts_waitcnt lgkmcnt(0)"
            : "=&v"(x[0]), "=&v"(x[1]), "=&v"(x[2]), "=&v"(x[3]), "=&v"(x[4]), "=&v"(x[5]), "=&v"(x[6]), "=&v"(x[7]), "=&v"(fx[0]),
              "=&v"(fx[1]), "=&v"(fx[2]), "=&v"(fx[3]), "=&v"(fx[4]), "=&v"(fx[5]), "=&v"(fx[6]), "=&v"(fx[7]), "=&v"(y[0]),
              "=&v"(y[1]), "=&v"(y[2]), "=&v"(y[3]), "=&v"(fw[0]), "=&v"(fw[1]), "=&v"(fw[2]), "=&v"(fw[3])
            : "v"(pa), "v"(pw), "v"(sa), "v"(sw)
            : "memory");
        if (part) settle();
        meet();
        __builtin_amdgcn_s_setprio(1);
#pragma unroll
        for (int t = 0; t < TN; ++t) {
          const i32x8 q = {(int)y[t][0], (int)y[t][1], (int)y[t][2], (int)y[t][3], 0, 0, 0, 0};
#pragma unroll
          for (int u = 0; u < TM; ++u) {
            const i32x8 v = {(int)x[u][0], (int)x[u][1], (int)x[u][2], (int)x[u][3], 0, 0, 0, 0};
            acc[t][u] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(q, v, acc[t][u], 4, 4, 0, (int)fw[t], 0, (int)fx[u]);
          }
        }
        __builtin_amdgcn_s_setprio(0);
        meet();
      }
    } else {
      uint32_t fw[TN];
#pragma unroll
      for (int part = 0; part < 2; ++part) {
        const uint32_t pa = address(slot + (wm * 128 + col) * 128 + (((quad ^ (col & 7)) ^ part * 4) * 16));
        const uint32_t pw = address(slot + kA + wn * 2048 + part * 512 + col * 16 + quad * 4);
        const uint32_t ps = address(sc + (wn * 64 + col) * 16 + (stage & 7) * 2);
        u32x4 x[TM];
        uint32_t w[TN];
        if (part == 0)
          asm volatile(
              "ds_read_u16 %12, %18\n\tds_read_u16 %13, %18 offset:256\n\tds_read_u16 %14, %18 offset:512\n\t"
              "ds_read_u16 %15, %18 offset:768\n\tds_read_b32 %8, %17\n\tds_read_b32 %9, %17 offset:256\n\t"
              "ds_read_b32 %10, %17 offset:1024\n\tds_read_b32 %11, %17 offset:1280\n\t"
              "ds_read_b128 %0, %16\n\tds_read_b128 %1, %16 offset:2048\n\tds_read_b128 %2, %16 offset:4096\n\t"
              "ds_read_b128 %3, %16 offset:6144\n\tds_read_b128 %4, %16 offset:8192\n\tds_read_b128 %5, %16 offset:10240\n\t"
              "ds_read_b128 %6, %16 offset:12288\n\tds_read_b128 %7, %16 offset:14336\n\ts_waitcnt lgkmcnt(0)"
              : "=&v"(x[0]), "=&v"(x[1]), "=&v"(x[2]), "=&v"(x[3]), "=&v"(x[4]), "=&v"(x[5]), "=&v"(x[6]), "=&v"(x[7]), "=&v"(w[0]),
                "=&v"(w[1]), "=&v"(w[2]), "=&v"(w[3]), "=&v"(fw[0]), "=&v"(fw[1]), "=&v"(fw[2]), "=&v"(fw[3])
              : "v"(pa), "v"(pw), "v"(ps)
              : "memory");
        else
          asm volatile(
              "ds_read_b32 %8, %13\n\tds_read_b32 %9, %13 offset:256\n\tds_read_b32 %10, %13 offset:1024\n\t"
              "ds_read_b32 %11, %13 offset:1280\n\t"
              "ds_read_b128 %0, %12\n\tds_read_b128 %1, %12 offset:2048\n\tds_read_b128 %2, %12 offset:4096\n\t"
              "ds_read_b128 %3, %12 offset:6144\n\tds_read_b128 %4, %12 offset:8192\n\tds_read_b128 %5, %12 offset:10240\n\t"
              "ds_read_b128 %6, %12 offset:12288\n\tds_read_b128 %7, %12 offset:14336\n\ts_waitcnt lgkmcnt(0)"
              : "=&v"(x[0]), "=&v"(x[1]), "=&v"(x[2]), "=&v"(x[3]), "=&v"(x[4]), "=&v"(x[5]), "=&v"(x[6]), "=&v"(x[7]), "=&v"(w[0]),
                "=&v"(w[1]), "=&v"(w[2]), "=&v"(w[3])
              : "v"(pa), "v"(pw)
              : "memory");
        if constexpr (EXACT) {
          if (part == 1) settle();
          meet();
#pragma unroll
          for (int t = 0; t < TN; ++t) {
            const bf16x8 v = quarters_bf16(w[t], __builtin_bit_cast(float, fw[t] << (23 - 8 * part)));
#pragma unroll
            for (int u = 0; u < TM; ++u) acc[t][u] = times_exact(v, __builtin_bit_cast(f16x8, x[u]), acc[t][u]);
          }
        } else {
          f16x8 v[TN];
#pragma unroll
          for (int t = 0; t < TN; ++t) {
            v[t] = eight_f16(w[t], __builtin_bit_cast(float, fw[t] << (23 - 8 * part)));
            // factors of 2^-15 to 1, as weights have them, both parts' at a time
            if (part == 0) *far |= (fw[t] ^ 0x7070u) & 0xF0F0u;
            asm volatile("" : "+v"(v[t]));  // before the meeting, not behind it
          }
          if (part == 1) settle();
          meet();
          __builtin_amdgcn_s_setprio(1);
#pragma unroll
          for (int t = 0; t < TN; ++t)
#pragma unroll
            for (int u = 0; u < TM; ++u)
              acc[t][u] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v[t], __builtin_bit_cast(f16x8, x[u]), acc[t][u], 0, 0, 0);
          __builtin_amdgcn_s_setprio(0);
        }
        meet();
      }
    }
  }

  template <bool EXACT>
  __device__ __forceinline__ uint32_t sum(f32x4 (&acc)[TN][TM]) const {
    uint32_t far = 0;
#pragma unroll
    for (int t = 0; t < TN; ++t)
#pragma unroll
      for (int u = 0; u < TM; ++u) acc[t][u] = f32x4{};
    const int stages = (g.k + kDepth - 1) / kDepth;
    load_scales(0);
    // stages behind the last are loaded, too, as zeros: a wait counts the same loads always
#pragma unroll
    for (int i = 0; i < kRing - 1; ++i) load<true>(i, i);
    wait<(kRing - 2) * kLoads>();
    meet();
    if (wave >= 4) meet();
    int at = 0;
#pragma unroll 1
    for (int s = 0; s < stages; ++s) {
      const int next = s + kRing - 1, free = at == 0 ? kRing - 1 : at - 1;
      if (s % kSpan == 0) load_scales(s / kSpan + 1);
      if (next < stages - 1)
        load<false>(free, next);
      else
        load<true>(free, next);
      multiply<EXACT>(at, s, &far, acc);
      at = at + 1 == kRing ? 0 : at + 1;
    }
    if (wave < 4) meet();
    wait<0>();
    meet();
    return far;
  }
  // Whether f16 does not hold a weight of the tile: factors one by one.
  __device__ __forceinline__ bool outside() const {
    bool odd = false;
    for (int i = threadIdx.x; i < blocks * kRowsW; i += 512) {
      const size_t r = min(n0 + i / blocks, g.n - 1), b = i % blocks;
      if (g.ws[r * g.pitch + b] - 104u > 36u) {
        const uint4 q = *(const uint4*)(g.w + (r * blocks + b) * 16);
        odd |= ((q.x | q.y | q.z | q.w) & 0x77777777u) != 0;
      }
    }
    return odd;
  }
};

}  // namespace

}  // namespace dw
