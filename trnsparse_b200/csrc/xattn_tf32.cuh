// fp32 attention products on the tensor cores: m16n8k8 tf32 with both operands split in two (3xTF32).
//
// x = hi + lo with hi the nearest tf32 value (11 bits) and lo the rest cut to 11 bits; a b ~ lo_a hi_b + hi_a lo_b +
// hi_a hi_b. |lo| <= 2^-11 |x| and lo loses at most 2^-23 |x|, so a product is off by less than 2^-22 + 2 * 2^-23 =
// 2^-21 of |a b|, eight half steps of fp32; sums are fp32. Values are finite (the rest of an infinity is not a number).
// The tf32 form does 510 multiply-adds a clock and SM here, 170 after the split, against 128 of the CUDA cores at
// best and 60 as attention kernels on them got: a warp's B operand is one 4-byte read a lane where they read
// 16 bytes for every four multiply-adds.
//
// Layouts (lane = 4 g + t): A (16 x 8) rows g, g + 8, columns t, t + 4; B (8 x 8) rows t, t + 4, column g; C rows g,
// g + 8, columns 2 t, 2 t + 1. A score tile's C becomes the A of the next product without an exchange: its columns
// 2 t, 2 t + 1 are taken as the contraction indexes t, t + 4, and B's rows are read in that order.
#pragma once

#include "xattn_tc.cuh"

namespace tsb {
namespace {

__device__ __forceinline__ void split_tf32(float x, uint32_t& hi, uint32_t& lo) {
  // nearest, halves away from zero, in two integer operations
  hi = (__float_as_uint(x) + 0x1000u) & 0xffffe000u;
  lo = __float_as_uint(x - __uint_as_float(hi)) & 0xffffe000u;
}
// Not volatile: the products of different tiles are independent, and the compiler may interleave them.
__device__ __forceinline__ void mma_tf32(float (&c)[4], const uint32_t (&a)[4], const uint32_t (&b)[2]) {
  asm("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, "
      "%3};\n"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b[0]), "r"(b[1]));
}
// c[m][n0 + n] += a[m] b[n], b0 and b1 this lane's two elements of tile n
template <int MT, int N, int NC>
__device__ __forceinline__ void mma_3xtf32(float (&c)[MT][NC][4], int n0, const uint32_t (&ah)[MT][4],
                                           const uint32_t (&al)[MT][4], const float (&b0)[N], const float (&b1)[N]) {
  uint32_t bh[N][2], bl[N][2];
#pragma unroll
  for (int n = 0; n < N; ++n) {
    split_tf32(b0[n], bh[n][0], bl[n][0]);
    split_tf32(b1[n], bh[n][1], bl[n][1]);
  }
#pragma unroll
  for (int i = 0; i < 3; ++i)
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int n = 0; n < N; ++n) mma_tf32(c[m][n0 + n], i ? ah[m] : al[m], i == 1 ? bl[n] : bh[n]);
}

// c[m][n] += F X^T over the first D columns: F the warp's 16 MT rows, X the 8 NT walked rows (both DP floats apart).
template <int MT, int NT, int DP>
__device__ __forceinline__ void scores_tf32(float (&c)[MT][NT][4], const float* F, const float* X, int D, int g, int t) {
#pragma unroll (MT == 1 ? 2 : 1)
  for (int k = 0; k < D; k += 8) {
    float b0[NT], b1[NT];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      b0[n] = X[(n * 8 + g) * DP + k + t];
      b1[n] = X[(n * 8 + g) * DP + k + t + 4];
    }
    uint32_t ah[MT][4], al[MT][4];
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      const float* f = F + (m * 16 + g) * DP + k + t;
      split_tf32(f[0], ah[m][0], al[m][0]);
      split_tf32(f[8 * DP], ah[m][1], al[m][1]);
      split_tf32(f[4], ah[m][2], al[m][2]);
      split_tf32(f[8 * DP + 4], ah[m][3], al[m][3]);
    }
    mma_3xtf32<MT, NT, NT>(c, 0, ah, al, b0, b1);
  }
}

// acc[m] += P X: P the scores' tiles (16 MT x 8 NT), X the walked rows, NO tiles of 8 columns.
template <int MT, int NT, int NO, int DP>
__device__ __forceinline__ void weigh_tf32(float (&acc)[MT][NO][4], const float (&p)[MT][NT][4], const float* X, int g,
                                           int t) {
  constexpr int STEP = MT == 1 ? 8 : 4;
#pragma unroll
  for (int k = 0; k < NT; ++k) {
    uint32_t ah[MT][4], al[MT][4];
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      split_tf32(p[m][k][0], ah[m][0], al[m][0]);
      split_tf32(p[m][k][2], ah[m][1], al[m][1]);
      split_tf32(p[m][k][1], ah[m][2], al[m][2]);
      split_tf32(p[m][k][3], ah[m][3], al[m][3]);
    }
    const float* x = X + (k * 8 + 2 * t) * DP + g;
#pragma unroll
    for (int n0 = 0; n0 < NO; n0 += STEP) {
      float b0[STEP], b1[STEP];
#pragma unroll
      for (int n = 0; n < STEP; ++n) {
        b0[n] = x[(n0 + n) * 8];
        b1[n] = x[DP + (n0 + n) * 8];
      }
      mma_3xtf32<MT, STEP, NO>(acc, n0, ah, al, b0, b1);
    }
  }
}

}  // namespace
}  // namespace tsb
