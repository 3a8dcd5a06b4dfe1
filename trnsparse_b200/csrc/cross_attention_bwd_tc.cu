// Backward of cross attention on the tensor cores (bf16 operands, fp32 sums;
// head_dim a multiple of 8 up to 128):
//   P = 2^(s2 - lse), dP = dO V^T, dS = P (dP - D), D = rowsum(dO o O),
//   dQ = scale dS K,  dK = scale dS^T Q,  dV = P^T dO   (dK, dV over the group's heads).
// P and dS are formed in fp32 and rounded to bf16 once, as operands of their
// products (half a step each, of the size of the results' own rounding: errors of
// 2.4e-3 of the gradients' size where that rounding alone makes 1.7e-3).
//
// Two launches of one kernel, each owning what it writes (fixed order, no
// atomics, seven products for the mathematics' five):
//   rows     fixed Q, dO of 128 query rows; walks the key tiles       -> dQ
//   columns  fixed K, V of 128 keys; walks the 128-row tiles of every
//            query head of the group                                  -> dK, dV
// A step multiplies two fixed tiles F1, F2 and two walked tiles X1, X2:
//   S = F1 X1^T, dP = F2 X2^T, acc0 += dS X1, and in columns acc1 += P X2.
// One CTA per SM, 10 warps: warp 8 TMA producer, warp 9 MMA issuer, warps 0-7
// the pointwise part (thread = TMEM lane warp % 4, 64 of the 128 columns). P
// and dS overwrite scores in TMEM (A operands of the second products), each half
// of the columns at the start of its own 64. MMAs run in issue order. Columns:
// acc1 += P_j X2_j, S_{j+1}, acc0 += dS_j X1_j, dP_{j+1}; rows, with two S
// buffers: dP_{j+1}, acc0 += dS_j X1_j, S_{j+2}.
//
// What bounds it: the chain of a step. At head_dim 128 a step of rows takes 2260
// clocks for 3 products of 512, one of columns 3320 for 4: the tensor pipe is busy 70
// and 63% of the time, and the rest is the pointwise part between the two products of
// a step (scores out of TMEM, 2^x, P and dS back), as deep as TMEM allows: rows have a
// second S, columns none, their 512 columns being S, dP, dK and dV. Loads are not
// waited for (walked tiles: 64 KB a step). 4 x 16 heads, 2048 x 4096 x 128: dQ 324 us
// and dK, dV 461 us, 1272 and 1192 TFLOP/s of their three and four products.
//
// Hidden keys: P and dS are set to zero by selection; in rows the K rows of
// hidden keys are zeroed in shared memory before dS K, so NaN in padding meets
// no product that is kept. In columns a hidden key is a lane of its own.
#include "xattn_tc.cuh"

namespace tsb {
namespace {

constexpr int kBwThreads = 320;

template <int HD, bool COL>
struct BwLayout {
  static constexpr int kChunks = HD / 64;
  static constexpr int kTile = 128 * HD * 2;
  static constexpr int kX1Stages = 3, kX2Stages = 2;
  static constexpr int kF1 = 0, kF2 = kTile, kX1 = 2 * kTile;
  static constexpr int kX2 = kX1 + kX1Stages * kTile;
  static constexpr int kStat = kX2 + kX2Stages * kTile;  // two stages: the walked rows' -log-sum-exp and -D
  static constexpr int kBar = kStat + 2 * 1024;
  static constexpr int kSmem = kBar + 256;
  // columns: S / P, dP / dS, dK, dV; rows: two S / dS, dP, dQ
  static constexpr uint32_t kTmemS = 0, kTmemDP = COL ? 128 : 256, kTmemAcc0 = COL ? 256 : 384, kTmemAcc1 = 384;
};

struct BwBars {
  uint64_t f_full, f_empty, x1_full[3], x1_empty[3], x2_full[2], x2_empty[2], st_full[2], st_empty[2];
  uint64_t s_full[2], dp_full, p_half, p_full, ds_full, acc_full;
  uint32_t tmem_slot;
  int abort_flag;
};

struct BwArgs {
  const int* lengths;
  const uint8_t* mask;
  int64_t mask_stride;
  const float *nlse, *ndelta;  // -log-sum-exp and -D, [batch, q_heads, padded tokens]
  void *out0, *out1;         // dQ, or dK and dV
  int64_t s0[3], s1[3];      // their strides
  float *part0, *part1;      // fp32 parts [parts][rows][D], or null
  int64_t part_rows;
  int Hq, Hkv, G, Sq, Sk, D, q_tiles, k_tiles, parts, chunk;
  int mul_h[4], mul_b[4];    // q, dout, k, v
  float scale, scale_log2;
};

__device__ __forceinline__ int bw_len(const BwArgs& A, int b) {
  return A.lengths == nullptr ? A.Sk : max(0, min(A.lengths[b], A.Sk));
}

// Unit u: part p of the walk of a fixed tile; b outermost, so round-robin CTAs see every length alike.
struct BwUnit {
  int b, h, tile, part, beg, end;  // h: query head (rows) or key head (columns)
  int rot;                         // the walk starts `rot` steps behind beg and wraps
  __device__ int step(int i) const {
    const int s = beg + rot + i;
    return s < end ? s : s - (end - beg);
  }
};
template <bool COL>
__device__ __forceinline__ BwUnit bw_unit(const BwArgs& A, int u) {
  const int heads = COL ? A.Hkv : A.Hq, tiles = COL ? A.k_tiles : A.q_tiles;
  BwUnit x;
  x.part = u % A.parts;
  u /= A.parts;
  x.tile = u % tiles;
  u /= tiles;
  x.h = u % heads;
  x.b = u / heads;
  const int len = bw_len(A, x.b);
  const int steps = COL ? (x.tile * 128 < len ? A.G * A.q_tiles : 0) : (len + 127) / 128;
  x.beg = min(steps, x.part * A.chunk);
  x.end = min(steps, x.beg + A.chunk);
  // CTAs that run together share a head: each starts elsewhere in the walk, so they do not all read one tile
  // from the same few L2 slices at a time.
  x.rot = x.end > x.beg ? (x.tile * 5) % (x.end - x.beg) : 0;
  return x;
}

template <int HD, bool COL>
__global__ void __launch_bounds__(kBwThreads, 1)
xattn_bwd_tc_kernel(const __grid_constant__ CUtensorMap tq, const __grid_constant__ CUtensorMap tg,
                    const __grid_constant__ CUtensorMap tk, const __grid_constant__ CUtensorMap tv,
                    const __grid_constant__ BwArgs A, int units) {
  using Lay = BwLayout<HD, COL>;
  extern __shared__ __align__(16) uint8_t sb[];  // no static shared memory: 1024-byte aligned
  BwBars& B = *reinterpret_cast<BwBars*>(sb + Lay::kBar);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    mbar_init(&B.f_full, 1);
    mbar_init(&B.f_empty, 1);
    for (int i = 0; i < 3; ++i) {
      mbar_init(&B.x1_full[i], 1);
      mbar_init(&B.x1_empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&B.x2_full[i], 1);
      mbar_init(&B.x2_empty[i], 1);
      mbar_init(&B.st_full[i], 1);
      mbar_init(&B.st_empty[i], 1);
    }
    mbar_init(&B.s_full[0], 1);
    mbar_init(&B.s_full[1], 1);
    mbar_init(&B.dp_full, 1);
    mbar_init(&B.p_half, 256);
    mbar_init(&B.p_full, 256);
    mbar_init(&B.ds_full, 256);
    mbar_init(&B.acc_full, 1);
    B.abort_flag = (smem_u32(sb) & 1023u) ? 1 : 0;
    if (B.abort_flag) record_device_error(DEVERR_SELFCHECK_SMEM);
    fence_mbar_init();
  }
  if (warp == 9) {
    tmem_alloc(&B.tmem_slot, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  grid_dep_wait();  // the row sums come from the kernel before
  const uint32_t tmem = B.tmem_slot;
  volatile int* abort_flag = &B.abort_flag;
  const int padded = A.q_tiles * 128;

  if (warp == 8) {
    // ---------------- producers: lane 0 the fixed tiles and X1, lane 1 X2, in columns lane 2 the statistics (rings
    // of their own: each is released at another time)
    if (lane < (COL ? 3 : 2) && !*abort_flag) {
      int n = 0, nu = 0;
      bool ok = true;
      for (int u = blockIdx.x; ok && u < units; u += gridDim.x) {
        const BwUnit x = bw_unit<COL>(A, u);
        if (x.beg >= x.end) continue;
        if (lane == 0) {
          if (nu > 0 && !mbar_wait(&B.f_empty, (nu - 1) & 1)) { ok = false; break; }
          mbar_arrive_expect_tx(&B.f_full, 2 * Lay::kTile);
          for (int c = 0; c < Lay::kChunks; ++c) {
            if (COL) {
              tma_load_4d(sb + Lay::kF1 + c * 16384, &tk, c * 64, x.tile * 128, x.h * A.mul_h[2], x.b * A.mul_b[2], &B.f_full);
              tma_load_4d(sb + Lay::kF2 + c * 16384, &tv, c * 64, x.tile * 128, x.h * A.mul_h[3], x.b * A.mul_b[3], &B.f_full);
            } else {
              tma_load_4d(sb + Lay::kF1 + c * 16384, &tq, c * 64, x.tile * 128, x.h * A.mul_h[0], x.b * A.mul_b[0], &B.f_full);
              tma_load_4d(sb + Lay::kF2 + c * 16384, &tg, c * 64, x.tile * 128, x.h * A.mul_h[1], x.b * A.mul_b[1], &B.f_full);
            }
          }
        }
        ++nu;
        for (int i = 0; i < x.end - x.beg; ++i, ++n) {
          const int s = x.step(i);
          int h, row;
          if (COL) {
            const int g = s / A.q_tiles;
            h = x.h * A.G + g;
            row = (s - g * A.q_tiles) * 128;
          } else {
            h = x.h / A.G;
            row = s * 128;
          }
          if (lane == 0) {
            const int st = n % Lay::kX1Stages, use = n / Lay::kX1Stages;
            if (*abort_flag || (use > 0 && !mbar_wait(&B.x1_empty[st], (use - 1) & 1))) { ok = false; break; }
            uint8_t* dst = sb + Lay::kX1 + st * Lay::kTile;
            mbar_arrive_expect_tx(&B.x1_full[st], Lay::kTile);
            constexpr int w = COL ? 0 : 2;
            for (int c = 0; c < Lay::kChunks; ++c)
              tma_load_4d(dst + c * 16384, COL ? &tq : &tk, c * 64, row, h * A.mul_h[w], x.b * A.mul_b[w], &B.x1_full[st]);
          } else if (lane == 1) {
            const int st = n % Lay::kX2Stages, use = n / Lay::kX2Stages;
            if (*abort_flag || (use > 0 && !mbar_wait(&B.x2_empty[st], (use - 1) & 1))) { ok = false; break; }
            uint8_t* dst = sb + Lay::kX2 + st * Lay::kTile;
            mbar_arrive_expect_tx(&B.x2_full[st], Lay::kTile);
            constexpr int w = COL ? 1 : 3;
            for (int c = 0; c < Lay::kChunks; ++c)
              tma_load_4d(dst + c * 16384, COL ? &tg : &tv, c * 64, row, h * A.mul_h[w], x.b * A.mul_b[w], &B.x2_full[st]);
          } else {
            const int st = n & 1, use = n >> 1;
            if (*abort_flag || (use > 0 && !mbar_wait(&B.st_empty[st], (use - 1) & 1))) { ok = false; break; }
            uint8_t* dst = sb + Lay::kStat + st * 1024;
            const int64_t at = (static_cast<int64_t>(x.b) * A.Hq + h) * padded + row;
            mbar_arrive_expect_tx(&B.st_full[st], 1024);
            bulk_g2s(dst, A.nlse + at, 512, &B.st_full[st]);
            bulk_g2s(dst + 512, A.ndelta + at, 512, &B.st_full[st]);
          }
        }
      }
      if (!ok) {
        atomicExch(&B.abort_flag, 1);
        // copies in flight land before the CTA may end
        if (lane == 0) {
          if (nu > 0) mbar_wait(&B.f_full, (nu - 1) & 1);
          for (int i = max(0, n - Lay::kX1Stages); i < n; ++i)
            mbar_wait(&B.x1_full[i % Lay::kX1Stages], (i / Lay::kX1Stages) & 1);
        } else if (lane == 1) {
          for (int i = max(0, n - Lay::kX2Stages); i < n; ++i)
            mbar_wait(&B.x2_full[i % Lay::kX2Stages], (i / Lay::kX2Stages) & 1);
        } else {
          for (int i = max(0, n - 2); i < n; ++i) mbar_wait(&B.st_full[i & 1], (i >> 1) & 1);
        }
      }
    }
  } else if (warp == 9) {
    // ---------------- MMA issuer
    if (warp_all(!*abort_flag)) {
      constexpr uint32_t idesc_s = make_idesc(MmaKind::BF16, 128, 128);
      constexpr uint32_t idesc_a = make_idesc(MmaKind::BF16, 128, HD) | (1u << 16);  // walked tile MN-major
      const bool lead = elect_one();
      // descriptors are formed once and moved by adding to their address field (16-byte units)
      const uint64_t dk = smem_desc_sw128(smem_u32(sb + Lay::kF1)), dm = smem_desc_sw128_mn(smem_u32(sb + Lay::kF1), 16384);
      const uint32_t base = static_cast<uint32_t>(dk);
      constexpr uint32_t kF2 = (Lay::kF2 - Lay::kF1) >> 4, kX1 = (Lay::kX1 - Lay::kF1) >> 4, kX2 = (Lay::kX2 - Lay::kF1) >> 4;
      auto product = [&](uint32_t d, uint32_t f, uint32_t x, int kk) {
        const uint32_t off = ((kk >> 2) * 16384 + (kk & 3) * 32) >> 4;
        umma<MmaKind::BF16>(d, desc_at(dk, base + f + off), desc_at(dk, base + x + off), idesc_s, kk > 0);
      };
      // acc += A X with A packed in TMEM: columns 64 h .. of half h
      auto accumulate = [&](uint32_t acc, uint32_t a, uint32_t x, int kk, bool add) {
        umma_ts_f16(acc, a + (kk >> 2) * 64 + (kk & 3) * 8, desc_at(dm, static_cast<uint32_t>(dm) + x + kk * (2048 >> 4)),
                    idesc_a, add);
      };
      // ring positions of the current and the next step
      int s1 = 0, u1 = 0, s2 = 0, u2 = 0;
      auto next1 = [&] {
        if (++s1 == Lay::kX1Stages) {
          s1 = 0;
          ++u1;
        }
      };
      auto next2 = [&] {
        if (++s2 == Lay::kX2Stages) {
          s2 = 0;
          ++u2;
        }
      };
      auto x1_at = [&] { return kX1 + s1 * (Lay::kTile >> 4); };
      auto x2_at = [&] { return kX2 + s2 * (Lay::kTile >> 4); };
      auto ensure = [&](bool seen, uint64_t* bar, int parity) { return warp_all(seen || mbar_wait(bar, parity & 1)); };
      constexpr int kK = HD / 16;
      int n = 0, nu = 0;
      bool ok = true;
      for (int u = blockIdx.x; ok && u < units; u += gridDim.x) {
        const BwUnit x = bw_unit<COL>(A, u);
        const int steps = x.end - x.beg;
        if (steps <= 0) continue;
        if (!ensure(false, &B.f_full, nu)) { ok = false; break; }
        ++nu;
        // Barriers are looked at before the last MMA of a burst and waited for only if they were not complete then
        // (cross_attention_tc.cu).
        if constexpr (COL) {
          if (!ensure(false, &B.x1_full[s1], u1)) { ok = false; break; }
          tc_fence_after();
          if (lead) {
#pragma unroll
            for (int kk = 0; kk < kK; ++kk) product(tmem + Lay::kTmemS, 0, x1_at(), kk);
            umma_commit(&B.s_full[0]);
          }
          if (!ensure(false, &B.x2_full[s2], u2)) { ok = false; break; }
          if (lead) {
#pragma unroll
            for (int kk = 0; kk < kK; ++kk) product(tmem + Lay::kTmemDP, kF2, x2_at(), kk);
            umma_commit(&B.dp_full);
            if (steps == 1) umma_commit(&B.f_empty);
          }
          // s1, s2: this step's tiles
          bool p_seen = false;
          for (int j = 0; j < steps; ++j, ++n) {
            const bool more = j + 1 < steps;
            const uint32_t x1_now = x1_at(), x2_now = x2_at();
            const int e1 = s1, e2 = s2;
            next1();
            next2();
            auto pv = [&](int kk, bool add) { accumulate(tmem + Lay::kTmemAcc1, tmem + Lay::kTmemS, x2_now, kk, add); };
            // P of the first 32 columns of each warp half (k-steps 0, 1, 4, 5), then the rest
            if (!ensure(p_seen, &B.p_half, n)) { ok = false; break; }
            tc_fence_after();
            if (lead) {
              pv(0, j > 0);
              pv(1, true);
              pv(4, true);
            }
            const bool f_seen = mbar_test_wait(&B.p_full, n & 1);
            if (lead) pv(5, true);
            if (!ensure(f_seen, &B.p_full, n)) { ok = false; break; }
            tc_fence_after();
            bool x1_seen = !more, ds_seen = false, x2_seen = !more;
            if (lead) {
              pv(2, true);
              pv(3, true);
              pv(6, true);
            }
            if (more) x1_seen = mbar_test_wait(&B.x1_full[s1], u1 & 1);
            else ds_seen = mbar_test_wait(&B.ds_full, n & 1);
            if (lead) {
              pv(7, true);
              umma_commit(&B.x2_empty[e2]);
            }
            if (more) {
              if (!ensure(x1_seen, &B.x1_full[s1], u1)) { ok = false; break; }
#pragma unroll
              for (int kk = 0; kk < kK - 1; ++kk)
                if (lead) product(tmem + Lay::kTmemS, 0, x1_at(), kk);
              ds_seen = mbar_test_wait(&B.ds_full, n & 1);
              if (lead) {
                product(tmem + Lay::kTmemS, 0, x1_at(), kK - 1);
                umma_commit(&B.s_full[0]);
              }
            }
            if (!ensure(ds_seen, &B.ds_full, n)) { ok = false; break; }
            tc_fence_after();
#pragma unroll
            for (int kk = 0; kk < 7; ++kk)
              if (lead) accumulate(tmem + Lay::kTmemAcc0, tmem + Lay::kTmemDP, x1_now, kk, j > 0 || kk > 0);
            if (more) x2_seen = mbar_test_wait(&B.x2_full[s2], u2 & 1);
            if (lead) {
              accumulate(tmem + Lay::kTmemAcc0, tmem + Lay::kTmemDP, x1_now, 7, true);
              umma_commit(&B.x1_empty[e1]);
              umma_commit(&B.st_empty[n & 1]);  // ds_full: the pointwise warps are through with them
            }
            if (more) {
              if (!ensure(x2_seen, &B.x2_full[s2], u2)) { ok = false; break; }
#pragma unroll
              for (int kk = 0; kk < kK - 1; ++kk)
                if (lead) product(tmem + Lay::kTmemDP, kF2, x2_at(), kk);
              p_seen = mbar_test_wait(&B.p_half, (n + 1) & 1);
              if (lead) {
                product(tmem + Lay::kTmemDP, kF2, x2_at(), kK - 1);
                umma_commit(&B.dp_full);
                if (j + 2 == steps) umma_commit(&B.f_empty);  // the last use of the fixed tiles
              }
            } else if (lead) {
              umma_commit(&B.acc_full);
            }
          }
        } else {
          // Rows need no P in TMEM, which leaves room for two S: S runs a step ahead of the pointwise warps, dS goes
          // over the S it came from, and the next dP is issued before dS K: no product waits for a pointwise step
          // but the one that needs its result.
          if (!ensure(false, &B.x1_full[s1], u1)) { ok = false; break; }
          tc_fence_after();
          int c1 = s1;  // this step's K; s1 runs ahead to the next S
          auto next_s = [&](int m) {
            if (lead) {
#pragma unroll
              for (int kk = 0; kk < kK; ++kk) product(tmem + Lay::kTmemS + (m & 1) * 128, 0, x1_at(), kk);
              umma_commit(&B.s_full[m & 1]);
            }
            next1();
          };
          next_s(n);
          if (!ensure(false, &B.x2_full[s2], u2)) { ok = false; break; }
          if (lead) {
#pragma unroll
            for (int kk = 0; kk < kK; ++kk) product(tmem + Lay::kTmemDP, kF2, x2_at(), kk);
            umma_commit(&B.dp_full);
            umma_commit(&B.x2_empty[s2]);
            if (steps == 1) umma_commit(&B.f_empty);
          }
          next2();
          if (steps > 1) {
            if (!ensure(false, &B.x1_full[s1], u1)) { ok = false; break; }
            next_s(n + 1);
          }
          bool ds_seen = false;
          for (int j = 0; j < steps; ++j, ++n) {
            const bool more = j + 1 < steps;
            bool x2_seen = more && mbar_test_wait(&B.x2_full[s2], u2 & 1);
            if (!ensure(ds_seen, &B.ds_full, n)) { ok = false; break; }
            ds_seen = false;
            tc_fence_after();
            if (more) {
              if (!ensure(x2_seen, &B.x2_full[s2], u2)) { ok = false; break; }
              if (lead) {
#pragma unroll
                for (int kk = 0; kk < kK; ++kk) product(tmem + Lay::kTmemDP, kF2, x2_at(), kk);
                umma_commit(&B.dp_full);
                umma_commit(&B.x2_empty[s2]);
                if (j + 2 == steps) umma_commit(&B.f_empty);  // the last use of the fixed tiles
              }
              next2();
            }
            const uint32_t x1_now = kX1 + c1 * (Lay::kTile >> 4);
#pragma unroll
            for (int kk = 0; kk < 7; ++kk)
              if (lead) accumulate(tmem + Lay::kTmemAcc0, tmem + Lay::kTmemS + (n & 1) * 128, x1_now, kk, j > 0 || kk > 0);
            const bool x1_seen = j + 2 < steps && mbar_test_wait(&B.x1_full[s1], u1 & 1);
            if (lead) {
              accumulate(tmem + Lay::kTmemAcc0, tmem + Lay::kTmemS + (n & 1) * 128, x1_now, 7, true);
              umma_commit(&B.x1_empty[c1]);
              if (!more) umma_commit(&B.acc_full);
            }
            c1 = c1 + 1 == Lay::kX1Stages ? 0 : c1 + 1;
            if (j + 2 < steps) {
              if (!ensure(x1_seen, &B.x1_full[s1], u1)) { ok = false; break; }
              if (lead) {
#pragma unroll
                for (int kk = 0; kk < kK; ++kk) product(tmem + Lay::kTmemS + (n & 1) * 128, 0, x1_at(), kk);
                umma_commit(&B.s_full[n & 1]);
              }
              next1();
              ds_seen = mbar_test_wait(&B.ds_full, (n + 1) & 1);
            }
          }
        }
      }
      if (!ok && lead) atomicExch(&B.abort_flag, 1);
    }
  } else {
    // ---------------- pointwise part: lane = fixed row, 64 columns a thread
    const int half = warp >> 2, r = threadIdx.x & 127;
    const uint32_t lane_base = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t t_s = tmem + Lay::kTmemS + lane_base + half * 64, t_dp = tmem + Lay::kTmemDP + lane_base + half * 64;
    const uint64_t sl2 = pack2(A.scale_log2, A.scale_log2);
    int n = 0, nu = 0;
    bool ok = warp_all(!*abort_flag);
    for (int u = blockIdx.x; ok && u < units; u += gridDim.x) {
      const BwUnit x = bw_unit<COL>(A, u);
      const int len = bw_len(A, x.b);
      const uint8_t* mask = A.mask ? A.mask + x.b * A.mask_stride : nullptr;
      const int fixed = x.tile * 128 + r;
      uint64_t row_nlse = 0, row_ndelta = 0;
      bool dead = false;  // columns: this key is hidden
      if (COL) {
        dead = fixed >= len || (mask && !mask[fixed]);
      } else {
        const int64_t at = (static_cast<int64_t>(x.b) * A.Hq + x.h) * padded + fixed;
        row_nlse = pack2(A.nlse[at], A.nlse[at]);
        row_ndelta = pack2(A.ndelta[at], A.ndelta[at]);
      }
      const bool any_dead = COL && __any_sync(0xffffffffu, dead);
      for (int step = 0; step < x.end - x.beg; ++step, ++n) {
        const int s = x.step(step);
        uint32_t kept[2] = {~0u, ~0u};
        bool part = false;
        if (!COL) {
          part = mask != nullptr || s * 128 + 128 > len;
          if (part) {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              const int key = s * 128 + half * 64 + 32 * i + lane;
              kept[i] = __ballot_sync(0xffffffffu, key < len && (mask == nullptr || mask[key] != 0));
            }
          }
        }
        const float* st = reinterpret_cast<const float*>(sb + Lay::kStat + (n & 1) * 1024) + half * 64;
        if (!warp_all(!*abort_flag && mbar_wait(&B.s_full[COL ? 0 : n & 1], (COL ? n : n >> 1) & 1))) { ok = false; break; }
        if (COL && !warp_all(mbar_wait(&B.st_full[n & 1], (n >> 1) & 1))) { ok = false; break; }
        tc_fence_after();
        const uint32_t t_sn = t_s + (COL ? 0 : (n & 1) * 128);
        uint32_t p[2][32], pk[32];
        tmem_ld32(t_sn, p[0]);
        tmem_ld32(t_sn + 32, p[1]);
        tmem_wait_ld32(p[0]);
        tmem_wait_ld32(p[1]);
        // hidden keys: the packed P and dS become zeros, whatever was computed
        auto hide = [&](uint32_t* w, int c) {
          if (COL) {
            if (any_dead)
#pragma unroll
              for (int i = 0; i < 16; ++i) w[i] = dead ? 0u : w[i];
          } else if (part) {
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              const uint32_t k = kept[c] >> (2 * i);
              w[i] &= (k & 1u ? 0xffffu : 0u) | (k & 2u ? 0xffff0000u : 0u);
            }
          }
        };
        // Packed fp32 arithmetic; one in four exponentials on the FMA pipe (two warps of a scheduler share a
        // special-function unit that does four a clock).
#pragma unroll
        for (int c = 0; c < 2; ++c) {
#pragma unroll
          for (int i = 0; i < 32; i += 4) {
            uint64_t l0 = row_nlse, l1 = row_nlse;
            if (COL) {
              const ulonglong2 ls = *reinterpret_cast<const ulonglong2*>(st + c * 32 + i);
              l0 = ls.x;
              l1 = ls.y;
            }
            const uint64_t x0 = fma2(pack2(__uint_as_float(p[c][i]), __uint_as_float(p[c][i + 1])), sl2, l0);
            const uint64_t x1 = fma2(pack2(__uint_as_float(p[c][i + 2]), __uint_as_float(p[c][i + 3])), sl2, l1);
            float e0, e1, e2, e3;
            unpack2(x0, e0, e1);
            e0 = ex2(e0);
            e1 = ex2(e1);
            if (i % 8 == 4) {
              exp2_poly2(x1, e2, e3);
            } else {
              unpack2(x1, e2, e3);
              e2 = ex2(e2);
              e3 = ex2(e3);
            }
            p[c][i] = __float_as_uint(e0);
            p[c][i + 1] = __float_as_uint(e1);
            p[c][i + 2] = __float_as_uint(e2);
            p[c][i + 3] = __float_as_uint(e3);
            if (COL) {
              pk[c * 16 + i / 2] = pack_bf16(e0, e1);
              pk[c * 16 + i / 2 + 1] = pack_bf16(e2, e3);
            }
          }
          if (COL) {
            hide(pk + c * 16, c);
            tmem_st16(t_s + c * 16, pk + c * 16);
            tmem_wait_st();
            tc_fence_before();
            mbar_arrive(c ? &B.p_full : &B.p_half);
          }
        }
        if (!COL && part && half == 0) {
          // hidden keys' K rows become zeros before dS K (their scores are read already)
          const int key = s * 128 + r;
          if (!(key < len && (mask == nullptr || mask[key] != 0))) {
            uint8_t* kr = sb + Lay::kX1 + (n % Lay::kX1Stages) * Lay::kTile + r * 128;
#pragma unroll
            for (int c = 0; c < Lay::kChunks; ++c)
#pragma unroll
              for (int q = 0; q < 8; ++q) *reinterpret_cast<uint4*>(kr + c * 16384 + q * 16) = make_uint4(0u, 0u, 0u, 0u);
          }
          fence_proxy_async_smem();
        }
        if (!warp_all(mbar_wait(&B.dp_full, n & 1))) { ok = false; break; }
        tc_fence_after();
        uint32_t dp[2][32];
        tmem_ld32(t_dp, dp[0]);
        tmem_wait_ld32(dp[0]);
        tmem_ld32(t_dp + 32, dp[1]);
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          if (c) tmem_wait_ld32(dp[1]);
#pragma unroll
          for (int i = 0; i < 32; i += 4) {
            uint64_t d0 = row_ndelta, d1 = row_ndelta;
            if (COL) {
              const ulonglong2 de = *reinterpret_cast<const ulonglong2*>(st + 128 + c * 32 + i);
              d0 = de.x;
              d1 = de.y;
            }
            const uint64_t t0 = mul2(pack2(__uint_as_float(p[c][i]), __uint_as_float(p[c][i + 1])),
                                     add2(pack2(__uint_as_float(dp[c][i]), __uint_as_float(dp[c][i + 1])), d0));
            const uint64_t t1 = mul2(pack2(__uint_as_float(p[c][i + 2]), __uint_as_float(p[c][i + 3])),
                                     add2(pack2(__uint_as_float(dp[c][i + 2]), __uint_as_float(dp[c][i + 3])), d1));
            float e0, e1, e2, e3;
            unpack2(t0, e0, e1);
            unpack2(t1, e2, e3);
            pk[c * 16 + i / 2] = pack_bf16(e0, e1);
            pk[c * 16 + i / 2 + 1] = pack_bf16(e2, e3);
          }
        }
        hide(pk, 0);
        hide(pk + 16, 1);
        tmem_st32(COL ? t_dp : t_sn, pk);
        tmem_wait_st();
        tc_fence_before();
        mbar_arrive(&B.ds_full);
      }
      if (!ok) break;
      // ---- accumulators -> global; a unit without steps writes zeros
      const bool worked = x.beg < x.end;
      if (worked) {
        if (!warp_all(mbar_wait(&B.acc_full, nu & 1) && !*abort_flag)) { ok = false; break; }
        ++nu;
        tc_fence_after();
      }
      const int limit = COL ? A.Sk : A.Sq;
      const bool live = fixed < limit;
      const int64_t fr = (static_cast<int64_t>(x.b) * (COL ? A.Hkv : A.Hq) + x.h) * (COL ? A.Sk : A.Sq) + fixed;
#pragma unroll
      for (int a = 0; a < (COL ? 2 : 1); ++a) {
        const int64_t* os = a ? A.s1 : A.s0;
        const float f = a ? 1.f : A.scale;
        float* po = a ? A.part1 : A.part0;
        __nv_bfloat16* ob = static_cast<__nv_bfloat16*>(a ? A.out1 : A.out0) + x.b * os[0] + x.h * os[1] + fixed * os[2];
        if (po != nullptr) po += (static_cast<int64_t>(x.part) * A.part_rows + fr) * A.D;
#pragma unroll 1
        for (int c = 0; c < HD / 64; ++c) {  // half h: columns h HD / 2 ..
          const int d0 = half * (HD / 2) + c * 32;
          uint32_t v[32];
          if (worked) {
            tmem_ld32(tmem + (a ? Lay::kTmemAcc1 : Lay::kTmemAcc0) + lane_base + d0, v);
            tmem_wait_ld32(v);
          } else {
#pragma unroll
            for (int i = 0; i < 32; ++i) v[i] = 0u;
          }
          auto val = [&](int i) { return __uint_as_float(v[i]) * f; };
          if (live && po != nullptr) {
#pragma unroll
            for (int i = 0; i < 32; i += 4)
              if (d0 + i < A.D)
                *reinterpret_cast<float4*>(po + d0 + i) = make_float4(val(i), val(i + 1), val(i + 2), val(i + 3));
          } else if (po == nullptr) {
            // four lanes exchange their four 16-byte pieces, so that a store writes 64 contiguous bytes of a row
            uint4 q[4];
#pragma unroll
            for (int i = 0; i < 4; ++i)
              q[i] = make_uint4(pack_bf16(val(8 * i), val(8 * i + 1)), pack_bf16(val(8 * i + 2), val(8 * i + 3)),
                                pack_bf16(val(8 * i + 4), val(8 * i + 5)), pack_bf16(val(8 * i + 6), val(8 * i + 7)));
            quad_transpose(q, lane & 3);
            const int d = d0 + (lane & 3) * 8;
#pragma unroll
            for (int k = 0; k < 4; ++k)
              if (fixed - (lane & 3) + k < limit && d < A.D)
                *reinterpret_cast<uint4*>(ob + (k - (lane & 3)) * os[2] + d) = q[k];
          }
        }
      }
      tc_fence_before();  // the accumulators are read before the next unit's first product (ordered by p_full, ds_full)
    }
    if (!ok) atomicExch(&B.abort_flag, 1);
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (warp == 9) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// -D = -rowsum(dO o O) and the log-sum-exp negated, padded to whole 128-row tiles (-inf there: P = 0). 16 lanes a
// row. Negated, they enter the packed multiply-adds as they are.
__global__ void __launch_bounds__(256) xattn_row_sums_kernel(const __nv_bfloat16* __restrict__ dout,
                                                             const __nv_bfloat16* __restrict__ out,
                                                             const float* __restrict__ lse, int64_t rows, int Hq,
                                                             int Sq, int padded, int D, int64_t g_b, int64_t g_h,
                                                             int64_t g_t, int64_t o_b, int64_t o_h, int64_t o_t,
                                                             float* nlse, float* ndelta) {
  grid_dep_launch();
  const int64_t row = static_cast<int64_t>(blockIdx.x) * 16 + (threadIdx.x >> 4);
  const int c = threadIdx.x & 15;
  const bool in = row < rows;
  const int64_t bh = in ? row / padded : 0;
  const int t = in ? static_cast<int>(row - bh * padded) : 0;
  float s = 0.f;
  if (in && t < Sq && c * 8 < D) {
    const int64_t b = bh / Hq, h = bh - b * Hq;
    const uint4 g = *reinterpret_cast<const uint4*>(dout + b * g_b + h * g_h + t * g_t + c * 8);
    const uint4 o = *reinterpret_cast<const uint4*>(out + b * o_b + h * o_h + t * o_t + c * 8);
    const uint32_t gw[4] = {g.x, g.y, g.z, g.w}, ow[4] = {o.x, o.y, o.z, o.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      s = fmaf(__uint_as_float(gw[i] << 16), __uint_as_float(ow[i] << 16), s);
      s = fmaf(__uint_as_float(gw[i] & 0xffff0000u), __uint_as_float(ow[i] & 0xffff0000u), s);
    }
  }
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  if (in && c == 0) {
    ndelta[row] = -s;
    nlse[row] = t < Sq ? -lse[bh * Sq + t] : -INFINITY;
  }
}

// out[b, h, t, :] = sum of the parts, in order; 8 elements a thread.
__global__ void __launch_bounds__(256) xattn_sum_bf16_kernel(const float* __restrict__ part, int parts, int64_t rows,
                                                             __nv_bfloat16* out, int H, int L, int D, int64_t o_b,
                                                             int64_t o_h, int64_t o_t) {
  const int64_t i = (static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x) * 8;
  if (i >= rows * D) return;
  const int64_t row = i / D;
  const int d = static_cast<int>(i - row * D);
  float s[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  for (int p = 0; p < parts; ++p) {
    const float4 a = *reinterpret_cast<const float4*>(part + p * rows * D + i);
    const float4 b = *reinterpret_cast<const float4*>(part + p * rows * D + i + 4);
    s[0] += a.x; s[1] += a.y; s[2] += a.z; s[3] += a.w;
    s[4] += b.x; s[5] += b.y; s[6] += b.z; s[7] += b.w;
  }
  const int64_t bh = row / L, t = row - bh * L, b = bh / H, h = bh - b * H;
  *reinterpret_cast<uint4*>(out + b * o_b + h * o_h + t * o_t + d) =
      make_uint4(pack_bf16(s[0], s[1]), pack_bf16(s[2], s[3]), pack_bf16(s[4], s[5]), pack_bf16(s[6], s[7]));
}

// Steps of an accumulator: the tensor core cuts what it adds to the accumulator's last place, and longer chains of one
// sign shrink visibly (kFwFlushTiles in cross_attention_tc.cu has the figures).
constexpr int64_t kBwMostSteps = 1024;

struct BwPlan {
  int q_tiles, k_tiles, parts[2], chunk[2], units[2];  // [0] rows, [1] columns
  size_t delta, part, total;
};

BwPlan bw_plan(const trnsparse_attention_args* a) {
  BwPlan p = {};
  const int sms = sm_count();
  const int64_t G = a->q_heads / a->kv_heads;
  p.q_tiles = static_cast<int>((a->q_len + 127) / 128);
  p.k_tiles = static_cast<int>((a->k_len + 127) / 128);
  const int64_t items[2] = {a->batch * a->q_heads * p.q_tiles, a->batch * a->kv_heads * p.k_tiles};
  const int64_t steps[2] = {p.k_tiles, G * p.q_tiles};
  const int64_t rows[2] = {a->batch * a->q_heads * a->q_len, 2 * a->batch * a->kv_heads * a->k_len};
  size_t part = 0;
  for (int i = 0; i < 2; ++i) {
    // cut the walks where tiles are fewer than SMs; a part is at least four steps and at most kBwMostSteps
    int64_t parts = items[i] > 0 ? sms / items[i] : 1;
    if (parts > steps[i] / 4) parts = steps[i] / 4;
    if (parts * kBwMostSteps < steps[i]) parts = (steps[i] + kBwMostSteps - 1) / kBwMostSteps;
    if (parts < 1) parts = 1;
    const int64_t chunk = steps[i] > 0 ? (steps[i] + parts - 1) / parts : 1;
    p.chunk[i] = static_cast<int>(chunk);
    p.parts[i] = static_cast<int>(steps[i] > 0 ? (steps[i] + chunk - 1) / chunk : 1);
    p.units[i] = static_cast<int>(items[i] * p.parts[i]);
    if (p.parts[i] > 1) {
      const size_t b = sizeof(float) * static_cast<size_t>(p.parts[i]) * rows[i] * a->head_dim;
      part = part > b ? part : b;
    }
  }
  const size_t stats = align256(sizeof(float) * a->batch * a->q_heads * p.q_tiles * 128);
  p.delta = stats;
  p.part = 2 * stats;
  p.total = p.part + part;
  return p;
}

template <int HD, bool COL>
int bw_launch(const BwArgs& A, const XMap (&m)[4], int units, cudaStream_t st) {
  using Lay = BwLayout<HD, COL>;
  auto kern = xattn_bwd_tc_kernel<HD, COL>;
  static unsigned long long done = 0;  // a bit per device; setting the attribute again is harmless
  int rc = allow_smem(kern, Lay::kSmem, &done, "cross_attention backward: set smem");
  if (rc) return rc;
  const int sms = sm_count();
  cudaError_t e = launch_pdl(kern, dim3(units < sms ? units : sms), dim3(kBwThreads), Lay::kSmem, st, m[0].map, m[1].map,
                 m[2].map, m[3].map, A, units);
  if (e != cudaSuccess) return cuda_status(e, "cross_attention backward launch");
  return debug_sync(st, COL ? "cross_attention backward: dK, dV" : "cross_attention backward: dQ");
}

int bw_sum(const float* part, int parts, int64_t rows, void* out, int H, int L, int D, const int64_t* os,
           cudaStream_t st) {
  const int64_t n = rows * D / 8;
  xattn_sum_bf16_kernel<<<static_cast<unsigned>((n + 255) / 256), 256, 0, st>>>(
      part, parts, rows, static_cast<__nv_bfloat16*>(out), H, L, D, os[0], os[1], os[2]);
  TSB_CHECK_LAUNCH("cross_attention backward: sum of parts");
  return TRNSPARSE_OK;
}

}  // namespace

bool xattn_bwd_tc_ok(const trnsparse_attention_args* a) {
  if (!xattn_tc_ok(a, false)) return false;
  const int64_t B = a->batch, Hq = a->q_heads, Hk = a->kv_heads, Sq = a->q_len, Sk = a->k_len;
  if (!aligned16(a->dout) || !strides_ok(a->dout_strides, B, Hq, Sq, true) ||
      !strides_ok(a->q_strides, B, Hq, Sq, true))
    return false;
  if (a->dq && (!aligned16(a->dq) || !strides_ok(a->dq_strides, B, Hq, Sq, false))) return false;
  if (a->dk && (!aligned16(a->dk) || !aligned16(a->dv) || !strides_ok(a->dk_strides, B, Hk, Sk, false) ||
                !strides_ok(a->dv_strides, B, Hk, Sk, false)))
    return false;
  // units and padded rows are counted in 31 bits
  const int64_t qt = (Sq + 127) / 128, kt = (Sk + 127) / 128;
  return B * Hq * qt < (1ll << 23) && B * Hk * kt < (1ll << 23) && (Hq / Hk) * qt < (1ll << 30);
}

size_t xattn_bwd_tc_workspace(const trnsparse_attention_args* a) { return bw_plan(a).total; }

int xattn_bwd_tc(const trnsparse_attention_args* a, void* ws, cudaStream_t st) {
  const BwPlan p = bw_plan(a);
  const int64_t B = a->batch, Hq = a->q_heads, Hk = a->kv_heads, Sq = a->q_len, Sk = a->k_len, D = a->head_dim;
  XMap m[4];
  const int64_t *qs = a->q_strides, *gs = a->dout_strides, *ks = a->k_strides, *vs = a->v_strides;
  int rc = make_xmap(&m[0], a->q, D, Sq, Hq, B, qs[2], qs[1], qs[0], 128);
  if (!rc) rc = make_xmap(&m[1], a->dout, D, Sq, Hq, B, gs[2], gs[1], gs[0], 128);
  if (!rc) rc = make_xmap(&m[2], a->k, D, Sk, Hk, B, ks[2], ks[1], ks[0], 128);
  if (!rc) rc = make_xmap(&m[3], a->v, D, Sk, Hk, B, vs[2], vs[1], vs[0], 128);
  if (rc) return rc;
  char* w = static_cast<char*>(ws);
  float *lse = reinterpret_cast<float*>(w), *delta = reinterpret_cast<float*>(w + p.delta);
  float* part = reinterpret_cast<float*>(w + p.part);
  const int64_t rows = B * Hq * p.q_tiles * 128;
  const int64_t* os = a->out_strides;
  xattn_row_sums_kernel<<<static_cast<unsigned>((rows + 15) / 16), 256, 0, st>>>(
      static_cast<const __nv_bfloat16*>(a->dout), static_cast<const __nv_bfloat16*>(a->out), a->lse, rows, (int)Hq,
      (int)Sq, p.q_tiles * 128, (int)D, gs[0], gs[1], gs[2], os[0], os[1], os[2], lse, delta);
  TSB_CHECK_LAUNCH("cross_attention backward: row sums");
  BwArgs A = {};
  A.lengths = a->key_lengths;
  A.mask = a->key_mask;
  A.mask_stride = a->key_mask_stride;
  A.nlse = lse;
  A.ndelta = delta;
  A.Hq = (int)Hq;
  A.Hkv = (int)Hk;
  A.G = (int)(Hq / Hk);
  A.Sq = (int)Sq;
  A.Sk = (int)Sk;
  A.D = (int)D;
  A.q_tiles = p.q_tiles;
  A.k_tiles = p.k_tiles;
  for (int i = 0; i < 4; ++i) {
    A.mul_h[i] = m[i].mul_h;
    A.mul_b[i] = m[i].mul_b;
  }
  A.scale = static_cast<float>(a->scale);
  A.scale_log2 = static_cast<float>(a->scale * 1.4426950408889634);
  if (a->dk) {
    A.out0 = a->dk;
    A.out1 = a->dv;
    for (int i = 0; i < 3; ++i) {
      A.s0[i] = a->dk_strides[i];
      A.s1[i] = a->dv_strides[i];
    }
    A.parts = p.parts[1];
    A.chunk = p.chunk[1];
    A.part_rows = B * Hk * Sk;
    A.part0 = A.parts > 1 ? part : nullptr;
    A.part1 = A.parts > 1 ? part + A.parts * A.part_rows * D : nullptr;
    rc = D <= 64 ? bw_launch<64, true>(A, m, p.units[1], st) : bw_launch<128, true>(A, m, p.units[1], st);
    if (!rc && A.parts > 1) rc = bw_sum(A.part0, A.parts, A.part_rows, a->dk, (int)Hk, (int)Sk, (int)D, a->dk_strides, st);
    if (!rc && A.parts > 1) rc = bw_sum(A.part1, A.parts, A.part_rows, a->dv, (int)Hk, (int)Sk, (int)D, a->dv_strides, st);
    if (rc) return rc;
  }
  if (a->dq) {
    A.out0 = a->dq;
    A.out1 = nullptr;
    for (int i = 0; i < 3; ++i) A.s0[i] = a->dq_strides[i];
    A.parts = p.parts[0];
    A.chunk = p.chunk[0];
    A.part_rows = B * Hq * Sq;
    A.part0 = A.parts > 1 ? part : nullptr;
    A.part1 = nullptr;
    rc = D <= 64 ? bw_launch<64, false>(A, m, p.units[0], st) : bw_launch<128, false>(A, m, p.units[0], st);
    if (!rc && A.parts > 1) rc = bw_sum(A.part0, A.parts, A.part_rows, a->dq, (int)Hq, (int)Sq, (int)D, a->dq_strides, st);
  }
  return rc;
}

}  // namespace tsb
