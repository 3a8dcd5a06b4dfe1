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
// c[m][n0 + n] += a[m][k] b[k][n] over K products of 8. The matrix unit cuts its sums instead of rounding them, which
// over a chain of a few hundred keys shrank the results by 4e-6: every K products start from zero, the small terms
// first, and are added to the sum by a rounded addition.
template <int MT, int K, int N, int NC, typename B>
__device__ __forceinline__ void mma_3xtf32(float (&c)[MT][NC][4], int n0, const uint32_t (&ah)[K][MT][4],
                                           const uint32_t (&al)[K][MT][4], B b) {
  float s[MT][N][4];
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int n = 0; n < N; ++n) s[m][n][0] = s[m][n][1] = s[m][n][2] = s[m][n][3] = 0.f;
#pragma unroll
  for (int k = 0; k < K; ++k) {
    uint32_t bh[N][2], bl[N][2];
#pragma unroll
    for (int n = 0; n < N; ++n) {
      const float2 v = b(k, n0 + n);
      split_tf32(v.x, bh[n][0], bl[n][0]);
      split_tf32(v.y, bh[n][1], bl[n][1]);
    }
#pragma unroll
    for (int i = 0; i < 3; ++i)
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int n = 0; n < N; ++n) mma_tf32(s[m][n], i ? ah[k][m] : al[k][m], i == 1 ? bl[n] : bh[n]);
  }
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int n = 0; n < N; ++n)
#pragma unroll
      for (int j = 0; j < 4; ++j) c[m][n0 + n][j] += s[m][n][j];
}

// c[m][n] += F X^T over the first D columns: F the warp's 16 MT rows, X the 8 NT walked rows (both DP floats apart, zero
// from column D to the next multiple of 16).
template <int MT, int NT, int DP>
__device__ __forceinline__ void scores_tf32(float (&c)[MT][NT][4], const float* F, const float* X, int D, int g, int t) {
  constexpr int STEP = NT < 4 ? NT : 4;
  const float* f0 = F + g * DP + t;
  const float* x0 = X + g * DP + t;
#pragma unroll 1
  for (int k0 = 0; k0 < D; k0 += 16, f0 += 16, x0 += 16) {
    uint32_t ah[2][MT][4], al[2][MT][4];
#pragma unroll
    for (int k = 0; k < 2; ++k)
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        const float* f = f0 + m * 16 * DP + k * 8;
        split_tf32(f[0], ah[k][m][0], al[k][m][0]);
        split_tf32(f[8 * DP], ah[k][m][1], al[k][m][1]);
        split_tf32(f[4], ah[k][m][2], al[k][m][2]);
        split_tf32(f[8 * DP + 4], ah[k][m][3], al[k][m][3]);
      }
#pragma unroll
    for (int n0 = 0; n0 < NT; n0 += STEP)
      mma_3xtf32<MT, 2, STEP, NT>(c, n0, ah, al, [&](int k, int n) {
        const float* x = x0 + n * 8 * DP + k * 8;
        return make_float2(x[0], x[4]);
      });
  }
}

// acc[m] += P X: P the scores' tiles (16 MT x 8 NT), X the walked rows, NO tiles of 8 columns.
template <int MT, int NT, int NO, int DP>
__device__ __forceinline__ void weigh_tf32(float (&acc)[MT][NO][4], const float (&p)[MT][NT][4], const float* X, int g,
                                           int t) {
  constexpr int STEP = 4;
  const float* x0 = X + 2 * t * DP + g;
#pragma unroll
  for (int k0 = 0; k0 < NT; k0 += 2) {
    uint32_t ah[2][MT][4], al[2][MT][4];
#pragma unroll
    for (int k = 0; k < 2; ++k)
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        split_tf32(p[m][k0 + k][0], ah[k][m][0], al[k][m][0]);
        split_tf32(p[m][k0 + k][2], ah[k][m][1], al[k][m][1]);
        split_tf32(p[m][k0 + k][1], ah[k][m][2], al[k][m][2]);
        split_tf32(p[m][k0 + k][3], ah[k][m][3], al[k][m][3]);
      }
#pragma unroll
    for (int n0 = 0; n0 < NO; n0 += STEP)
      mma_3xtf32<MT, 2, STEP, NO>(acc, n0, ah, al, [&](int k, int n) {
        const float* x = x0 + (k0 + k) * 8 * DP + n * 8;
        return make_float2(x[0], x[DP]);
      });
  }
}

}  // namespace
}  // namespace tsb
