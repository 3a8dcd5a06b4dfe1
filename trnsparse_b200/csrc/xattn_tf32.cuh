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
  // rounded by integer arithmetic: a conversion instruction an element would cost more than the products
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
// c[n] += a b[n], b0 and b1 this lane's two elements of tile n
template <int N>
__device__ __forceinline__ void mma_3xtf32(float (&c)[N][4], const uint32_t (&ah)[4], const uint32_t (&al)[4],
                                           const float (&b0)[N], const float (&b1)[N]) {
  uint32_t bh[N][2], bl[N][2];
#pragma unroll
  for (int n = 0; n < N; ++n) {
    split_tf32(b0[n], bh[n][0], bl[n][0]);
    split_tf32(b1[n], bh[n][1], bl[n][1]);
  }
#pragma unroll
  for (int n = 0; n < N; ++n) mma_tf32(c[n], al, bh[n]);
#pragma unroll
  for (int n = 0; n < N; ++n) mma_tf32(c[n], ah, bl[n]);
#pragma unroll
  for (int n = 0; n < N; ++n) mma_tf32(c[n], ah, bh[n]);
}

// c[n] += F X^T over the first D columns: F the warp's 16 rows, X the NT * 8 walked rows (both DP floats apart).
template <int NT, int DP>
__device__ __forceinline__ void scores_tf32(float (&c)[NT][4], const float* F, const float* X, int D, int g, int t) {
#pragma unroll 2
  for (int k = 0; k < D; k += 8) {
    uint32_t ah[4], al[4];
    split_tf32(F[g * DP + k + t], ah[0], al[0]);
    split_tf32(F[(g + 8) * DP + k + t], ah[1], al[1]);
    split_tf32(F[g * DP + k + t + 4], ah[2], al[2]);
    split_tf32(F[(g + 8) * DP + k + t + 4], ah[3], al[3]);
    float b0[NT], b1[NT];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      b0[n] = X[(n * 8 + g) * DP + k + t];
      b1[n] = X[(n * 8 + g) * DP + k + t + 4];
    }
    mma_3xtf32<NT>(c, ah, al, b0, b1);
  }
}

// acc[n] += P X: P the scores' tiles (16 x 8 NT), X the walked rows, NO tiles of 8 columns.
template <int NT, int NO, int DP>
__device__ __forceinline__ void weigh_tf32(float (&acc)[NO][4], const float (&p)[NT][4], const float* X, int g, int t) {
#pragma unroll
  for (int k = 0; k < NT; ++k) {
    uint32_t ah[4], al[4];
    split_tf32(p[k][0], ah[0], al[0]);
    split_tf32(p[k][2], ah[1], al[1]);
    split_tf32(p[k][1], ah[2], al[2]);
    split_tf32(p[k][3], ah[3], al[3]);
    const float* x = X + (k * 8 + 2 * t) * DP + g;
#pragma unroll
    for (int n0 = 0; n0 < NO; n0 += 8) {
      float b0[8], b1[8];
#pragma unroll
      for (int n = 0; n < 8; ++n) {
        b0[n] = x[(n0 + n) * 8];
        b1[n] = x[DP + (n0 + n) * 8];
      }
      mma_3xtf32<8>(reinterpret_cast<float(&)[8][4]>(acc[n0]), ah, al, b0, b1);
    }
  }
}

}  // namespace
}  // namespace tsb
