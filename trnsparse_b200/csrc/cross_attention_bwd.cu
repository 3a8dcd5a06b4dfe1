// Backward of cross attention for fp32 at any head_dim up to 256, and for the
// bf16 shapes the tcgen05 kernels do not take. With the forward's
// row log-sum-exp (base 2) and D = rowsum(dO o O):
//   P = 2^(s2 - lse),  dP = dO V^T,  dS = P (dP - D),
//   dQ = scale dS K,  dK = scale dS^T Q,  dV = P^T dO,
// dK and dV summed over the query heads that share the key head. Hidden keys
// give exact zeros: their K and V rows are loaded as zeros and their P is set
// to zero, whatever the padding holds; a row without keys (lse = -inf) has
// only hidden keys.
//
// Two walks side by side in one launch, each owning what it writes, so sums have
// one fixed order (no atomics): rows (dQ: a tile of packed query rows walks the
// keys) and columns (dK, dV: a tile of keys walks every query row of its group).
// Both recompute P: five products of the mathematics cost seven, which buys
// repeatable results and no traffic for dQ. Where tiles are fewer than SMs the
// walks are cut into parts whose fp32 sums a last kernel adds in order.
//
// What bounds it: the tensor cores' tf32 rate (3xTF32, xattn_tf32.cuh), with the tensor
// pipe 51% busy on two warps a scheduler; the rest goes to splitting operands and to waits
// inside a warp's chain of scores, P and sums. 2 x 16/16 heads, 1024 x 1024 x 64: 644 us,
// 47 TFLOP/s of the seven products (on the CUDA cores 1171 us); 16/4 heads at head_dim
// 128 1278 us (2440); 2 x 8/2 heads, 333 x 517 x 64, where a CTA an SM is all there is,
// 96 us (108 with four warps a CTA, two CTAs an SM; that took 584 at the first size: the
// eight-warp form is faster for small calls only, and taken for all). 255 registers; at
// head_dim up to 64 350 bytes a thread are spilled and 510 read back, above 128 350 and 480
// (fp32), in between none.
#include "xattn_tf32.cuh"

namespace tsb {
namespace {

__device__ __forceinline__ float bcvt(float v) { return v; }
__device__ __forceinline__ float bcvt(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T>
__device__ __forceinline__ void bstore(T* p, float v) {
  if constexpr (sizeof(T) == 4) *p = v;
  else *p = __float2bfloat16_rn(v);
}
template <typename T>
__device__ __forceinline__ float4 bload4(const T* row, int d, int D, bool vec) {
  if (vec && d + 3 < D) {
    if constexpr (sizeof(T) == 4) return *reinterpret_cast<const float4*>(row + d);
    const uint2 w = *reinterpret_cast<const uint2*>(row + d);
    return make_float4(__uint_as_float(w.x << 16), __uint_as_float(w.x & 0xffff0000u), __uint_as_float(w.y << 16),
                       __uint_as_float(w.y & 0xffff0000u));
  }
  float4 r = make_float4(0.f, 0.f, 0.f, 0.f);
  if (d < D) r.x = bcvt(row[d]);
  if (d + 1 < D) r.y = bcvt(row[d + 1]);
  if (d + 2 < D) r.z = bcvt(row[d + 2]);
  if (d + 3 < D) r.w = bcvt(row[d + 3]);
  return r;
}
// One of the two walks: a CTA each for `tiles` tiles of every item and `parts` ranges of the walked rows.
struct BWalk {
  int tiles, chunk, parts;
  unsigned ctas;       // 0: not wanted
  float *part0, *part1;  // fp32 parts (null: one part, written to the outputs)
};

struct BKernel {
  XSide s;  // o_*: strides of dq here
  const void* dout;
  int64_t g_b, g_h, g_t;  // dout strides
  const float *lse, *delta;
  void *dq, *dk, *dv;
  int64_t dk_s[3], dv_s[3];
  BWalk rows, cols;
  int64_t all_rows, all_keys;  // rows of one part
  int D, vec;
  float scale, scale_log2;
};

// D = rowsum(dO o O) of every (batch, head, token) row; one warp per row.
template <typename T>
__global__ void __launch_bounds__(256) xattn_delta_kernel(const T* __restrict__ dout, const T* __restrict__ out,
                                                          int64_t rows, int Hq, int Tq, int D, int64_t g_b,
                                                          int64_t g_h, int64_t g_t, int64_t o_b, int64_t o_h,
                                                          int64_t o_t, float* delta) {
  const int64_t row = static_cast<int64_t>(blockIdx.x) * 8 + (threadIdx.x >> 5);
  if (row >= rows) return;
  const int lane = threadIdx.x & 31, t = static_cast<int>(row % Tq);
  const int64_t bh = row / Tq, b = bh / Hq, h = bh - b * Hq;
  const T* g = dout + b * g_b + h * g_h + t * g_t;
  const T* o = out + b * o_b + h * o_h + t * o_t;
  float s = 0.f;
  for (int d = lane; d < D; d += 32) s = fmaf(bcvt(g[d]), bcvt(o[d]), s);
  s = warp_sum(s);
  if (lane == 0) delta[row] = s;
}

// Eight warps, two a scheduler, so that one's products cover the other's exponentials. Up to head_dim 64 a warp has 32
// fixed rows, so that each split of a walked element feeds two products, and half of the walked ones (the halves' sums
// are joined at the end); up to 128 16 rows, as 32 rows' sums would not fit in registers; both with the next walked rows
// copied behind the arithmetic. Above that, 64 rows (shared memory), which warps share in pairs: for dQ each has half
// the walked keys, for dK and dV one each.
template <int DC>
struct BShape {
  static constexpr int kThreads = 256, kTiles16 = DC == 1 ? 2 : 1, kRows = DC == 4 ? 64 : 128;
  static constexpr int kWalk = DC == 1 ? 64 : 32;  // walked rows a step
  static constexpr int kStages = DC == 4 ? 1 : 2, kStride = DC * 64 + 4;
  static constexpr int kSmem = 4 * (2 * kRows * kStride + kStages * 2 * (kWalk * kStride + kWalk));
};

template <typename T, int DC, bool COLS>
__device__ __forceinline__ void bwd_walk(const BKernel& A, const BWalk& W, unsigned cta, float* smb) {
  using S = BShape<DC>;
  constexpr int MT = S::kTiles16, BT = S::kRows, WT = S::kWalk, NT = S::kThreads, STAGES = S::kStages;
  constexpr bool HALF = DC == 1 || (!COLS && DC == 4);  // a warp takes half the walked rows
  constexpr int DP = S::kStride, WW = HALF ? WT / 2 : WT, NW = WW / 8, NO = DC * 8, CH = DC * 16;
  constexpr int XS = 2 * (WT * DP + WT);  // floats of a stage
  constexpr bool BOTH = COLS && DC != 4;
  float* F1 = smb;           // fixed: Q (rows) or K (columns)
  float* F2 = F1 + BT * DP;  // fixed: dO or V
  float* X = F2 + BT * DP;   // walked, a stage: K or Q, V or dO, then (columns) the queries' lse and delta
  const XSide& s = A.s;
  const int tid = threadIdx.x, lane = tid & 31, g = lane >> 2, t = lane & 3;
  const int f0 = (tid >> 5) % (BT / 16 / MT) * 16 * MT;  // this warp's fixed rows
  const bool upper = tid >= 128;
  const bool second = COLS && DC == 4 && upper;  // holds dV
  const int x0 = HALF && upper ? WW : 0;
  const unsigned line = cta / W.parts, part = cta - line * W.parts;
  const int item = line / W.tiles, tile = line - item * W.tiles;
  const int bi = item / s.hkv, h = item - bi * s.hkv;
  const int64_t R = side_rows(s), fix0 = static_cast<int64_t>(tile) * BT;
  const int D = A.D, len = side_len(s, bi);
  const T* qp = static_cast<const T*>(s.q) + bi * s.q_bi + static_cast<int64_t>(h) * s.G * s.q_h;
  const T* gp = static_cast<const T*>(A.dout) + bi * A.g_b + static_cast<int64_t>(h) * s.G * A.g_h;
  const T* kp = static_cast<const T*>(s.k) + bi * s.k_b + h * s.k_h;
  const T* vp = static_cast<const T*>(s.v) + bi * s.v_b + h * s.v_h;
  const int64_t stat0 = (static_cast<int64_t>(bi) * s.hkv + h) * s.G * s.T;  // flat row of packed row 0
  const uint8_t* mask = s.mask ? s.mask + bi * s.mask_stride : nullptr;
  const bool busy = fix0 + f0 < (COLS ? len : R);  // a warp without rows only copies
  // fp32 rows that start on 16 bytes are copied asynchronously, the others through registers
  const bool async = sizeof(T) == 4 && A.vec && D % 4 == 0;
  const int c_row = tid / CH, c_d = (tid % CH) * 4;  // this thread's first row and its columns
  auto copy4 = [&](float* dst, const T* row, bool in) {
    if (async) {
      in = in && c_d < D;
      cp_async16(dst + c_d, in ? row + c_d : static_cast<const T*>(s.q), in);
    } else {
      *reinterpret_cast<float4*>(dst + c_d) = in ? bload4(row, c_d, D, A.vec) : make_float4(0.f, 0.f, 0.f, 0.f);
    }
  };
  auto load_q = [&](float* q, float* go, int64_t r0, int n) {
    for (int row = c_row; row < n; row += NT / CH) {
      const bool in = r0 + row < R;
      const unsigned r = in ? static_cast<unsigned>(r0 + row) : 0u, hg = r / s.T, tt = r - hg * s.T;
      copy4(q + row * DP, qp + hg * s.q_h + tt * s.q_t, in);
      copy4(go + row * DP, gp + hg * A.g_h + tt * A.g_t, in);
    }
  };
  auto load_kv = [&](float* k, float* v, int k0, int n) {
    for (int row = c_row; row < n; row += NT / CH) {
      const int key = k0 + row;
      const bool in = key < len && (!mask || mask[key]);
      copy4(k + row * DP, kp + key * s.k_t, in);
      copy4(v + row * DP, vp + key * s.v_t, in);
    }
  };
  if (COLS) load_kv(F1, F2, tile * BT, BT);
  else load_q(F1, F2, fix0, BT);
  grid_dep_wait();  // the row sums
  float row_lse[MT][2], row_delta[MT][2];  // rows: of this lane's queries
  bool hide_row[MT][2];  // columns: this lane's keys
#pragma unroll
  for (int a = 0; a < MT; ++a)
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int64_t r = fix0 + f0 + a * 16 + g + 8 * i;
      row_lse[a][i] = INFINITY;  // rows past the last: P = 0
      row_delta[a][i] = 0.f;
      hide_row[a][i] = false;
      if (COLS) {
        hide_row[a][i] = r >= len || (mask && !mask[r]);
      } else if (r < R) {
        row_lse[a][i] = A.lse[stat0 + r];
        row_delta[a][i] = A.delta[stat0 + r];
      }
    }
  float acc0[MT][NO][4], acc1[MT][BOTH ? NO : 1][4];
#pragma unroll
  for (int a = 0; a < MT; ++a)
#pragma unroll
    for (int n = 0; n < NO; ++n)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        acc0[a][n][j] = 0.f;
        if constexpr (BOTH) acc1[a][n][j] = 0.f;
      }
  auto step = [&](const float* x, int64_t w) {
    const float *X1 = x + x0 * DP, *X2 = X1 + WT * DP;
    const float *st_lse = x + 2 * WT * DP + x0, *st_delta = st_lse + WT;
    w += x0;
    float sc[MT][NW][4], dp[MT][NW][4];  // scores, then P; dP, then dS: fixed rows by walked rows
#pragma unroll
    for (int a = 0; a < MT; ++a)
#pragma unroll
      for (int n = 0; n < NW; ++n)
#pragma unroll
        for (int j = 0; j < 4; ++j) sc[a][n][j] = dp[a][n][j] = 0.f;
    bool seen = true;  // rows: key w + lane
    if (!COLS && (mask || w + WW > len)) seen = lane < WW && w + lane < len && (!mask || mask[w + lane]);
    scores_tf32<MT, NW, DP>(sc, F1 + f0 * DP, X1, D, g, t);
    if (!second) scores_tf32<MT, NW, DP>(dp, F2 + f0 * DP, X2, D, g, t);
    const unsigned keep = COLS ? 0u : __ballot_sync(0xffffffffu, seen);
#pragma unroll
    for (int n = 0; n < NW; ++n)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int i = j >> 1, x = n * 8 + 2 * t + (j & 1);
        bool hide = !COLS && !(keep >> x & 1u);
#pragma unroll
        for (int a = 0; a < MT; ++a) {
          if (COLS) hide = hide_row[a][i];
          const float p =
              hide ? 0.f : ex2(fmaf(sc[a][n][j], A.scale_log2, -(COLS ? st_lse[x] : row_lse[a][i])));
          dp[a][n][j] = hide ? 0.f : p * (dp[a][n][j] - (COLS ? st_delta[x] : row_delta[a][i]));
          sc[a][n][j] = p;
        }
      }
    if constexpr (BOTH) weigh_tf32<MT, NW, NO, DP>(acc1, sc, X2, g, t);
    if (second) weigh_tf32<MT, NW, NO, DP>(acc0, sc, X2, g, t);
    else weigh_tf32<MT, NW, NO, DP>(acc0, dp, X1, g, t);
  };
  // a walk over keys stops at the kept length; a key tile with no kept key walks nothing
  const int64_t wend = COLS ? (fix0 < len ? R : 0) : len;
  const int64_t w0 = static_cast<int64_t>(part) * W.chunk;
  const int64_t w1 = wend < w0 + W.chunk ? wend : w0 + W.chunk;
  float stat[2];  // columns: lse and delta of query w + tid, on their way to a stage
  auto copy_walked = [&](float* x, int64_t w) {
    if (COLS) {
      load_q(x, x + WT * DP, w, WT);
      const bool in = tid < WT && w + tid < R;
      stat[0] = in ? A.lse[stat0 + w + tid] : INFINITY;  // rows past the last: P = 0
      stat[1] = in ? A.delta[stat0 + w + tid] : 0.f;
    } else {
      load_kv(x, x + WT * DP, static_cast<int>(w), WT);
    }
  };
  auto put_stats = [&](float* x) {
    if (COLS && tid < WT) {
      x[2 * WT * DP + tid] = stat[0];
      x[2 * WT * DP + WT + tid] = stat[1];
    }
  };
  if (STAGES == 2 && w0 < w1) {
    copy_walked(X, w0);
    put_stats(X);
  }
  int stage = 0;
  for (int64_t w = w0; w < w1; w += WT) {
    float* X1 = X + stage * XS;
    if (STAGES == 1) {
      __syncthreads();
      copy_walked(X1, w);
      put_stats(X1);
    }
    cp_async_wait_all();
    __syncthreads();  // this stage has landed and the other one is read
    const bool more = STAGES == 2 && w + WT < w1;
    stage = STAGES == 2 ? stage ^ 1 : 0;
    if (more) copy_walked(X + stage * XS, w + WT);
    if (busy) step(X1, w);
    if (more) put_stats(X + stage * XS);
  }
  if constexpr (HALF) {  // both halves' sums, through the fixed tiles
    cp_async_wait_all();  // a walk without steps has not waited for them
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 2; ++i) {
#pragma unroll
      for (int a = 0; a < MT; ++a)
#pragma unroll
        for (int n = 0; n < NO; ++n)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int at = (f0 + a * 16 + g + 8 * (j >> 1)) * DP + n * 8 + 2 * t + (j & 1);
            if (i == 0 && upper) {
              F1[at] = acc0[a][n][j];
              if constexpr (BOTH) F2[at] = acc1[a][n][j];
            }
            if (i == 1) {
              acc0[a][n][j] += F1[at];
              if constexpr (BOTH) acc1[a][n][j] += F2[at];
            }
          }
      if (i == 0) __syncthreads();
      if (i == 0 && upper) return;
    }
  }
#pragma unroll
  for (int a = 0; a < MT; ++a)
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int64_t r = fix0 + f0 + a * 16 + g + 8 * i;
      if (r >= (COLS ? static_cast<int64_t>(s.klen) : R)) continue;
      const int64_t fr = COLS ? (static_cast<int64_t>(bi) * s.hkv + h) * s.klen + r : stat0 + r;
      const int64_t at = (static_cast<int64_t>(part) * (COLS ? A.all_keys : A.all_rows) + fr) * D;
      const bool piece = W.part0 != nullptr;
      T *o0 = nullptr, *o1 = nullptr;
      if (!piece && COLS) {
        o0 = static_cast<T*>(A.dk) + bi * A.dk_s[0] + h * A.dk_s[1] + r * A.dk_s[2];
        o1 = static_cast<T*>(A.dv) + bi * A.dv_s[0] + h * A.dv_s[1] + r * A.dv_s[2];
      } else if (!piece) {
        o0 = static_cast<T*>(A.dq) + o_offset(s, bi, h, side_row(s, r));
      }
      auto put = [&](float* pp, T* o, int d, float v) {
        if (piece) pp[at + d] = v;
        else bstore(o + d, v);
      };
#pragma unroll
      for (int n = 0; n < NO; ++n)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const int d = n * 8 + 2 * t + j;
          if (d >= D) continue;
          if (second) put(W.part1, o1, d, acc0[a][n][2 * i + j]);
          else put(W.part0, o0, d, acc0[a][n][2 * i + j] * A.scale);
          if constexpr (BOTH) put(W.part1, o1, d, acc1[a][n][2 * i + j]);
        }
    }
}

// The columns' CTAs first: their steps are the longer ones.
template <typename T, int DC>
__global__ void __launch_bounds__(BShape<DC>::kThreads, 1) xattn_bwd_mma_kernel(const BKernel A) {
  extern __shared__ __align__(16) float smb[];
  if (blockIdx.x < A.cols.ctas) bwd_walk<T, DC, true>(A, A.cols, blockIdx.x, smb);
  else bwd_walk<T, DC, false>(A, A.rows, blockIdx.x - A.cols.ctas, smb);
}

// out[b, h, t, :] = sum of the parts, in order, for up to three tensors.
struct BSum {
  const float* part[3];
  void* out[3];
  int64_t rows[3], o[3][3];
  int parts[3], H[3], L[3], D;
};
template <typename T>
__global__ void __launch_bounds__(256) xattn_sum_parts_kernel(const BSum A) {
  int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  grid_dep_wait();
#pragma unroll
  for (int k = 0; k < 3; ++k) {
    const int64_t n = A.rows[k] * A.D;
    if (i >= 0 && i < n) {
      const int64_t row = i / A.D;
      const int d = static_cast<int>(i - row * A.D);
      float s = 0.f;
      for (int p = 0; p < A.parts[k]; ++p) s += A.part[k][p * n + i];
      const int64_t bh = row / A.L[k], t = row - bh * A.L[k], b = bh / A.H[k], h = bh - b * A.H[k];
      bstore(static_cast<T*>(A.out[k]) + b * A.o[k][0] + h * A.o[k][1] + t * A.o[k][2] + d, s);
    }
    i -= n;
  }
}

// ---------------------------------------------------------------- host side

struct BPlan {
  int dc, tiles[2], parts[2], chunk[2];  // [0] rows (dQ), [1] columns (dK, dV)
  size_t at[2], ws;                      // the parts' place in the workspace, behind the row sums
};

BPlan bwd_plan(const trnsparse_attention_args* a, const XSide& s) {
  BPlan p = {};
  p.dc = a->head_dim <= 64 ? 1 : a->head_dim <= 128 ? 2 : 4;
  const int64_t R = side_rows(s);
  const int64_t fixed[2] = {R, s.klen}, walk[2] = {s.klen, R};
  const int bt = p.dc == 4 ? BShape<4>::kRows : BShape<1>::kRows;
  const int64_t wt = p.dc == 1 ? BShape<1>::kWalk : BShape<2>::kWalk;
  const int64_t rows = a->batch * a->q_heads * a->q_len, keys = a->batch * a->kv_heads * a->k_len;
  p.ws = (sizeof(float) * static_cast<size_t>(rows) + 255) & ~static_cast<size_t>(255);
  for (int i = 0; i < 2; ++i) {
    p.tiles[i] = static_cast<int>((fixed[i] + bt - 1) / bt);
    const int64_t ctas = static_cast<int64_t>(p.tiles[i]) * s.nb * s.hkv, steps = (walk[i] + wt - 1) / wt;
    // both walks run side by side: three and four of the seven products. Half a step a part: 108 us against 133 with
    // a tenth at 2 x 8/2 heads, 333 x 517 x 64
    const int64_t per = walk_steps(ctas, steps, sm_count() * (3 + i) / 7, 1, 32, 0.5);
    p.chunk[i] = static_cast<int>(per * wt);
    p.parts[i] = static_cast<int>(steps > 0 ? (steps + per - 1) / per : 1);
    p.at[i] = p.ws;
    if (p.parts[i] > 1)
      p.ws += (sizeof(float) * static_cast<size_t>(p.parts[i]) * a->head_dim * (i ? 2 * keys : rows) + 255) &
              ~static_cast<size_t>(255);
  }
  return p;
}

template <typename T, int DC>
int bwd_launch(const BKernel& A, cudaStream_t st) {
  auto kern = xattn_bwd_mma_kernel<T, DC>;
  cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, BShape<DC>::kSmem);
  if (e != cudaSuccess) return cuda_status(e, "cross_attention backward: set smem");
  e = launch_pdl(kern, dim3(A.cols.ctas + A.rows.ctas), dim3(BShape<DC>::kThreads), BShape<DC>::kSmem, st, A);
  return e == cudaSuccess ? TRNSPARSE_OK : cuda_status(e, "cross_attention backward launch");
}

template <typename T>
int bwd_general(const trnsparse_attention_args* a, void* ws, cudaStream_t st) {
  XSide s[2];
  int n = 0;
  int rc = make_sides(a, false, s, &n);
  if (rc) return rc;
  const BPlan p = bwd_plan(a, s[0]);
  const int Hq = (int)a->q_heads, Hkv = (int)a->kv_heads, Tq = (int)a->q_len, D = (int)a->head_dim;
  const int64_t rows = a->batch * a->q_heads * a->q_len, keys = a->batch * a->kv_heads * a->k_len;
  float* delta = static_cast<float*>(ws);
  const int64_t *gs = a->dout_strides, *os = a->out_strides;
  BKernel A = {};
  A.s = s[0];
  A.s.o_bi = a->dq_strides[0];
  A.s.o_h = a->dq_strides[1];
  A.s.o_t = a->dq_strides[2];
  A.dout = a->dout;
  A.g_b = gs[0];
  A.g_h = gs[1];
  A.g_t = gs[2];
  A.lse = a->lse;
  A.delta = delta;
  A.dq = a->dq;
  A.dk = a->dk;
  A.dv = a->dv;
  for (int i = 0; i < 3; ++i) {
    A.dk_s[i] = a->dk_strides[i];
    A.dv_s[i] = a->dv_strides[i];
  }
  A.D = D;
  A.all_rows = rows;
  A.all_keys = keys;
  const uintptr_t m = a->dtype == TRNSPARSE_F32 ? 15 : 7;
  const uintptr_t bases = reinterpret_cast<uintptr_t>(a->q) | reinterpret_cast<uintptr_t>(a->k) |
                          reinterpret_cast<uintptr_t>(a->v) | reinterpret_cast<uintptr_t>(a->dout);
  int64_t strides = 0;
  for (int i = 0; i < 3; ++i) strides |= a->q_strides[i] | a->k_strides[i] | a->v_strides[i] | gs[i];
  A.vec = !(bases & m) && !(strides & 3);
  A.scale = static_cast<float>(a->scale);
  A.scale_log2 = static_cast<float>(a->scale * 1.4426950408889634);
  BSum sum = {};
  sum.D = D;
  for (int i = 0; i < 2; ++i) {
    if (i ? !a->dk || keys == 0 : !a->dq) continue;
    BWalk& w = i ? A.cols : A.rows;
    const int64_t ctas = static_cast<int64_t>(p.tiles[i]) * p.parts[i] * s[0].nb * s[0].hkv;
    TSB_REQUIRE(ctas < (1ll << 30), "cross_attention backward: too many tiles (%lld)", static_cast<long long>(ctas));
    w.tiles = p.tiles[i];
    w.chunk = p.chunk[i];
    w.parts = p.parts[i];
    w.ctas = static_cast<unsigned>(ctas);
    if (w.parts == 1) continue;
    w.part0 = reinterpret_cast<float*>(static_cast<char*>(ws) + p.at[i]);
    w.part1 = i ? w.part0 + w.parts * keys * D : nullptr;
    for (int k = i; k < 1 + 2 * i; ++k) {  // dq; dk and dv
      sum.part[k] = k == 2 ? w.part1 : w.part0;
      sum.out[k] = k == 0 ? a->dq : k == 1 ? a->dk : a->dv;
      sum.rows[k] = i ? keys : rows;
      sum.parts[k] = w.parts;
      sum.H[k] = i ? Hkv : Hq;
      sum.L[k] = i ? static_cast<int>(a->k_len) : Tq;
      for (int j = 0; j < 3; ++j) sum.o[k][j] = (k == 0 ? a->dq_strides : k == 1 ? a->dk_strides : a->dv_strides)[j];
    }
  }
  if (A.rows.ctas + A.cols.ctas == 0) return TRNSPARSE_OK;
  xattn_delta_kernel<T><<<static_cast<unsigned>((rows + 7) / 8), 256, 0, st>>>(
      static_cast<const T*>(a->dout), static_cast<const T*>(a->out), rows, Hq, Tq, D, gs[0], gs[1], gs[2], os[0], os[1],
      os[2], delta);
  TSB_CHECK_LAUNCH("cross_attention backward: row sums");
  rc = p.dc == 1 ? bwd_launch<T, 1>(A, st) : p.dc == 2 ? bwd_launch<T, 2>(A, st) : bwd_launch<T, 4>(A, st);
  const int64_t elements = (sum.rows[0] + sum.rows[1] + sum.rows[2]) * D;
  if (rc || elements == 0) return rc;
  cudaError_t e = launch_pdl(xattn_sum_parts_kernel<T>, dim3(static_cast<unsigned>((elements + 255) / 256)), dim3(256), 0,
                             st, sum);
  return e == cudaSuccess ? TRNSPARSE_OK : cuda_status(e, "cross_attention backward: sum of parts");
}

}  // namespace
}  // namespace tsb

using namespace tsb;

extern "C" size_t trnsparse_cross_attention_backward_workspace_size(const trnsparse_attention_args* a) {
  if (check_attention(a, "cross_attention backward") || a->batch * a->q_heads * a->q_len == 0) return 0;
  if (xattn_bwd_tc_ok(a)) return xattn_bwd_tc_workspace(a);
  XSide s[2];
  int n = 0;
  make_sides(a, false, s, &n);
  return bwd_plan(a, s[0]).ws;
}

extern "C" int trnsparse_cross_attention_backward(const trnsparse_attention_args* a, void* ws, size_t ws_bytes,
                                                  void* stream) {
  int rc = check_attention(a, "cross_attention backward");
  if (rc) return rc;
  TSB_REQUIRE(a->batch * a->q_heads * a->q_len > 0, "cross_attention backward: no query rows");
  TSB_REQUIRE(a->q && a->out && a->lse && a->dout && (a->k_len == 0 || (a->k && a->v && !a->dk == !a->dv)),
              "cross_attention backward: null pointer");
  const size_t need = trnsparse_cross_attention_backward_workspace_size(a);
  TSB_REQUIRE(ws && ws_bytes >= need, "cross_attention backward: workspace too small (%zu bytes, needs %zu)", ws_bytes,
              need);
  cudaStream_t st = as_stream(stream);
  if (xattn_bwd_tc_ok(a)) return xattn_bwd_tc(a, ws, st);
  return a->dtype == TRNSPARSE_F32 ? bwd_general<float>(a, ws, st) : bwd_general<__nv_bfloat16>(a, ws, st);
}
