// Backward of cross attention on CUDA cores (fp32 at any head_dim up to 256,
// and the bf16 shapes the tensor-core kernels do not take). With the forward's
// row log-sum-exp (base 2) and D = rowsum(dO o O):
//   P = 2^(s2 - lse),  dP = dO V^T,  dS = P (dP - D),
//   dQ = scale dS K,  dK = scale dS^T Q,  dV = P^T dO,
// dK and dV summed over the query heads that share the key head. Hidden keys
// give exact zeros: their K and V rows are loaded as zeros and their P is set
// to zero, whatever the padding holds; a row without keys (lse = -inf) has
// only hidden keys.
//
// Two kernels, each owning what it writes, so sums have one fixed order (no
// atomics): rows (dQ: a tile of packed query rows walks the keys) and columns
// (dK, dV: a tile of keys walks every query row of its group). Both recompute
// P: five products of the mathematics cost seven, which buys repeatable results
// and no traffic for dQ. fp32 FMA bounds both; tiles of 64 (32 above head_dim
// 128, where four 64-row tiles would not fit in shared memory) with RM x RM
// scores a thread. Where tiles are fewer than SMs the walk is cut into parts
// whose fp32 sums a last kernel adds in order.
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
constexpr int kBwdWalk = 32;  // walked rows a step

struct BKernel {
  XSide s;  // o_*: strides of dq here
  const void* dout;
  int64_t g_b, g_h, g_t;  // dout strides
  const float *lse, *delta;
  void *dq, *dk, *dv;
  int64_t dk_s[3], dv_s[3];
  float *part0, *part1;  // fp32 parts (null: one part, written to the outputs)
  int64_t rows_all;      // rows of one part
  int D, tiles, chunk, vec;
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

// 64 fixed rows (queries, or keys with COLS) a CTA, 16 a warp; WT walked rows a step. Above head_dim 128 the sums of
// dK and of dV have 128 registers a thread each: eight warps, the second four hold dV.
template <typename T, int DC, bool COLS>
__global__ void __launch_bounds__(COLS && DC == 4 ? 256 : 128, DC == 1 ? 4 : DC == 2 ? 2 : 1)
    xattn_bwd_mma_kernel(const BKernel A) {
  constexpr int BT = 64, WT = kBwdWalk, NT = COLS && DC == 4 ? 256 : 128;
  constexpr int DP = DC * 64 + 4, NW = WT / 8, NO = DC * 8, CH = DC * 16;
  constexpr bool BOTH = COLS && DC != 4;
  extern __shared__ __align__(16) float smb[];
  float* F1 = smb;             // fixed: Q (rows) or K (columns)
  float* F2 = F1 + BT * DP;    // fixed: dO or V
  float* X1 = F2 + BT * DP;    // walked: K or Q
  float* X2 = X1 + WT * DP;    // walked: V or dO
  float* st_lse = X2 + WT * DP;  // of the walked queries (columns)
  float* st_delta = st_lse + WT;
  const XSide& s = A.s;
  const int tid = threadIdx.x, g = (tid & 31) >> 2, t = tid & 3;
  const int f0 = (tid >> 5 & 3) * 16;                // this warp's fixed rows
  const bool second = COLS && DC == 4 && tid >= 128;  // holds dV
  const int item = blockIdx.x / A.tiles, tile = blockIdx.x - item * A.tiles;
  const int bi = item / s.hkv, h = item - bi * s.hkv;
  const int64_t R = side_rows(s);
  const int D = A.D, len = side_len(s, bi);
  const T* qp = static_cast<const T*>(s.q) + bi * s.q_bi + static_cast<int64_t>(h) * s.G * s.q_h;
  const T* gp = static_cast<const T*>(A.dout) + bi * A.g_b + static_cast<int64_t>(h) * s.G * A.g_h;
  const T* kp = static_cast<const T*>(s.k) + bi * s.k_b + h * s.k_h;
  const T* vp = static_cast<const T*>(s.v) + bi * s.v_b + h * s.v_h;
  const int64_t stat0 = (static_cast<int64_t>(bi) * s.hkv + h) * s.G * s.T;  // flat row of packed row 0
  const uint8_t* mask = s.mask ? s.mask + bi * s.mask_stride : nullptr;
  // fp32 rows that start on 16 bytes are copied asynchronously, the others through registers
  const bool async = sizeof(T) == 4 && A.vec && D % 4 == 0;
  auto copy4 = [&](float* dst, const T* row, int d, bool in) {
    if (async) {
      cp_async16(dst, in && d < D ? row + d : static_cast<const T*>(s.q), in && d < D);
    } else {
      *reinterpret_cast<float4*>(dst) = in ? bload4(row, d, D, A.vec) : make_float4(0.f, 0.f, 0.f, 0.f);
    }
  };
  auto load_q = [&](float* q, float* go, int64_t r0, int n) {
    for (int i = tid; i < n * CH; i += NT) {
      const int row = i / CH, d = (i - row * CH) * 4;
      const bool in = r0 + row < R;
      const unsigned r = in ? static_cast<unsigned>(r0 + row) : 0u, hg = r / s.T, tt = r - hg * s.T;
      copy4(q + row * DP + d, qp + hg * s.q_h + tt * s.q_t, d, in);
      copy4(go + row * DP + d, gp + hg * A.g_h + tt * A.g_t, d, in);
    }
  };
  auto load_kv = [&](float* k, float* v, int k0, int n) {
    for (int i = tid; i < n * CH; i += NT) {
      const int row = i / CH, d = (i - row * CH) * 4, key = k0 + row;
      const bool in = key < len && (!mask || mask[key]);
      copy4(k + row * DP + d, kp + key * s.k_t, d, in);
      copy4(v + row * DP + d, vp + key * s.v_t, d, in);
    }
  };
  if (COLS) load_kv(F1, F2, tile * BT, BT);
  else load_q(F1, F2, static_cast<int64_t>(tile) * BT, BT);
  float row_lse[2], row_delta[2];  // rows: of this lane's queries
  bool hide_row[2];                // columns: this lane's keys
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int64_t r = static_cast<int64_t>(tile) * BT + f0 + g + 8 * i;
    row_lse[i] = INFINITY;  // rows past the last: P = 0
    row_delta[i] = 0.f;
    hide_row[i] = false;
    if (COLS) {
      hide_row[i] = r >= len || (mask && !mask[r]);
    } else if (r < R) {
      row_lse[i] = A.lse[stat0 + r];
      row_delta[i] = A.delta[stat0 + r];
    }
  }
  float acc0[NO][4], acc1[BOTH ? NO : 1][4];
#pragma unroll
  for (int n = 0; n < NO; ++n)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      acc0[n][j] = 0.f;
      if constexpr (BOTH) acc1[n][j] = 0.f;
    }
  // a walk over keys stops at the kept length; a key tile with no kept key walks nothing
  const int64_t wend = COLS ? (tile * BT < len ? R : 0) : len;
  const int64_t w0 = static_cast<int64_t>(blockIdx.y) * A.chunk;
  const int64_t w1 = wend < w0 + A.chunk ? wend : w0 + A.chunk;
  for (int64_t w = w0; w < w1; w += WT) {
    __syncthreads();
    if (COLS) {
      load_q(X1, X2, w, WT);
      if (tid < WT) {
        const bool in = w + tid < R;
        st_lse[tid] = in ? A.lse[stat0 + w + tid] : INFINITY;
        st_delta[tid] = in ? A.delta[stat0 + w + tid] : 0.f;
      }
    } else {
      load_kv(X1, X2, static_cast<int>(w), WT);
    }
    cp_async_wait_all();
    __syncthreads();
    float sc[NW][4], dp[NW][4];  // scores, then P; dP, then dS: fixed rows by walked rows
#pragma unroll
    for (int n = 0; n < NW; ++n)
#pragma unroll
      for (int j = 0; j < 4; ++j) sc[n][j] = dp[n][j] = 0.f;
    scores_tf32<NW, DP>(sc, F1 + f0 * DP, X1, D, g, t);
    if (!second) scores_tf32<NW, DP>(dp, F2 + f0 * DP, X2, D, g, t);
#pragma unroll
    for (int n = 0; n < NW; ++n)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int i = j >> 1, x = n * 8 + 2 * t + (j & 1);
        bool hide = hide_row[i];
        if (!COLS) hide = w + x >= len || (mask && !mask[w + x]);
        const float p = hide ? 0.f : exp2f(fmaf(sc[n][j], A.scale_log2, -(COLS ? st_lse[x] : row_lse[i])));
        dp[n][j] = hide ? 0.f : p * (dp[n][j] - (COLS ? st_delta[x] : row_delta[i]));
        sc[n][j] = p;
      }
    if constexpr (BOTH) weigh_tf32<NW, NO, DP>(acc1, sc, X2, g, t);
    if (second) weigh_tf32<NW, NO, DP>(acc0, sc, X2, g, t);
    else weigh_tf32<NW, NO, DP>(acc0, dp, X1, g, t);
  }
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int64_t r = static_cast<int64_t>(tile) * BT + f0 + g + 8 * i;
    if (r >= (COLS ? static_cast<int64_t>(s.klen) : R)) continue;
    const int64_t fr = COLS ? (static_cast<int64_t>(bi) * s.hkv + h) * s.klen + r : stat0 + r;
    const int64_t at = (static_cast<int64_t>(blockIdx.y) * A.rows_all + fr) * D;
    const bool piece = A.part0 != nullptr;
    T *o0 = nullptr, *o1 = nullptr;
    if (!piece && COLS) {
      o0 = static_cast<T*>(A.dk) + bi * A.dk_s[0] + h * A.dk_s[1] + r * A.dk_s[2];
      o1 = static_cast<T*>(A.dv) + bi * A.dv_s[0] + h * A.dv_s[1] + r * A.dv_s[2];
    } else if (!piece) {
      o0 = static_cast<T*>(A.dq) + o_offset(s, bi, h, side_row(s, r));
    }
    auto put = [&](float* part, T* o, int d, float v) {
      if (piece) part[at + d] = v;
      else bstore(o + d, v);
    };
#pragma unroll
    for (int n = 0; n < NO; ++n)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int d = n * 8 + 2 * t + j;
        if (d >= D) continue;
        if (second) put(A.part1, o1, d, acc0[n][2 * i + j]);
        else put(A.part0, o0, d, acc0[n][2 * i + j] * A.scale);
        if constexpr (BOTH) put(A.part1, o1, d, acc1[n][2 * i + j]);
      }
  }
}

// out[b, h, t, :] = sum of the parts, in order.
template <typename T>
__global__ void __launch_bounds__(256) xattn_sum_parts_kernel(const float* __restrict__ part, int parts, int64_t rows,
                                                              T* out, int H, int L, int D, int64_t o_b, int64_t o_h,
                                                              int64_t o_t) {
  const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (i >= rows * D) return;
  const int64_t row = i / D;
  const int d = static_cast<int>(i - row * D);
  float s = 0.f;
  for (int p = 0; p < parts; ++p) s += part[p * rows * D + i];
  const int64_t bh = row / L, t = row - bh * L, b = bh / H, h = bh - b * H;
  bstore(out + b * o_b + h * o_h + t * o_t + d, s);
}

// ---------------------------------------------------------------- host side

struct BPlan {
  int dc, parts[2], chunk[2], tiles[2];  // [0] rows (dQ), [1] columns (dK, dV)
  size_t ws;
};

BPlan bwd_plan(const trnsparse_attention_args* a, const XSide& s) {
  BPlan p = {};
  p.dc = a->head_dim <= 64 ? 1 : a->head_dim <= 128 ? 2 : 4;
  const int64_t R = side_rows(s);
  const int64_t fixed[2] = {R, s.klen}, walk[2] = {s.klen, R};
  const int64_t slots = (p.dc == 1 ? 4ll : p.dc == 2 ? 2ll : 1ll) * sm_count();  // resident CTAs
  const int64_t rows = a->batch * a->q_heads * a->q_len, keys = a->batch * a->kv_heads * a->k_len;
  p.ws = sizeof(float) * static_cast<size_t>(rows);
  size_t parts_ws = 0;
  for (int i = 0; i < 2; ++i) {
    p.tiles[i] = static_cast<int>((fixed[i] + 63) / 64);
    const int64_t ctas = static_cast<int64_t>(p.tiles[i]) * s.nb * s.hkv, steps = (walk[i] + kBwdWalk - 1) / kBwdWalk;
    const int64_t per = walk_steps(ctas, steps, slots, 32);
    p.chunk[i] = static_cast<int>(per * kBwdWalk);
    p.parts[i] = static_cast<int>(steps > 0 ? (steps + per - 1) / per : 1);
    if (p.parts[i] > 1) {
      const size_t b = sizeof(float) * static_cast<size_t>(p.parts[i]) * a->head_dim * (i ? 2 * keys : rows);
      parts_ws = parts_ws > b ? parts_ws : b;  // rows and columns run one after the other
    }
  }
  p.ws = ((p.ws + 255) & ~static_cast<size_t>(255)) + parts_ws;
  return p;
}

template <typename T, int DC, bool COLS>
int bwd_launch(const BKernel& A, int parts, cudaStream_t st) {
  constexpr size_t smem = sizeof(float) * (2ull * (64 + kBwdWalk) * (DC * 64 + 4) + 2 * kBwdWalk);
  auto kern = xattn_bwd_mma_kernel<T, DC, COLS>;
  cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem));
  if (e != cudaSuccess) return cuda_status(e, "cross_attention backward: set smem");
  const int threads = COLS && DC == 4 ? 256 : 128;
  if (A.tiles > 0)
    kern<<<dim3(static_cast<unsigned>(A.tiles) * A.s.nb * A.s.hkv, parts), threads, smem, st>>>(A);
  TSB_CHECK_LAUNCH("cross_attention backward launch");
  return TRNSPARSE_OK;
}

template <typename T, bool COLS>
int bwd_dispatch(const BKernel& A, int dc, int parts, cudaStream_t st) {
  if (dc == 1) return bwd_launch<T, 1, COLS>(A, parts, st);
  if (dc == 2) return bwd_launch<T, 2, COLS>(A, parts, st);
  return bwd_launch<T, 4, COLS>(A, parts, st);
}

template <typename T>
int sum_parts(const float* part, int parts, int64_t rows, void* out, int H, int L, int D, const int64_t* os,
              cudaStream_t st) {
  const int64_t n = rows * D;
  xattn_sum_parts_kernel<T><<<static_cast<unsigned>((n + 255) / 256), 256, 0, st>>>(
      part, parts, rows, static_cast<T*>(out), H, L, D, os[0], os[1], os[2]);
  TSB_CHECK_LAUNCH("cross_attention backward: sum of parts");
  return TRNSPARSE_OK;
}

template <typename T>
int bwd_simt(const trnsparse_attention_args* a, void* ws, cudaStream_t st) {
  XSide s[2];
  int n = 0;
  int rc = make_sides(a, false, s, &n);
  if (rc) return rc;
  const BPlan p = bwd_plan(a, s[0]);
  const int Hq = (int)a->q_heads, Hkv = (int)a->kv_heads, Tq = (int)a->q_len, D = (int)a->head_dim;
  const int64_t rows = a->batch * a->q_heads * a->q_len, keys = a->batch * a->kv_heads * a->k_len;
  float* delta = static_cast<float*>(ws);
  float* part = reinterpret_cast<float*>(static_cast<char*>(ws) +
                                         ((sizeof(float) * static_cast<size_t>(rows) + 255) & ~static_cast<size_t>(255)));
  const int64_t *gs = a->dout_strides, *os = a->out_strides;
  xattn_delta_kernel<T><<<static_cast<unsigned>((rows + 7) / 8), 256, 0, st>>>(
      static_cast<const T*>(a->dout), static_cast<const T*>(a->out), rows, Hq, Tq, D, gs[0], gs[1], gs[2], os[0], os[1],
      os[2], delta);
  TSB_CHECK_LAUNCH("cross_attention backward: row sums");
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
  const uintptr_t m = a->dtype == TRNSPARSE_F32 ? 15 : 7;
  const uintptr_t bases = reinterpret_cast<uintptr_t>(a->q) | reinterpret_cast<uintptr_t>(a->k) |
                          reinterpret_cast<uintptr_t>(a->v) | reinterpret_cast<uintptr_t>(a->dout);
  int64_t strides = 0;
  for (int i = 0; i < 3; ++i) strides |= a->q_strides[i] | a->k_strides[i] | a->v_strides[i] | gs[i];
  A.vec = !(bases & m) && !(strides & 3);
  A.scale = static_cast<float>(a->scale);
  A.scale_log2 = static_cast<float>(a->scale * 1.4426950408889634);

  A.tiles = p.tiles[0];
  A.chunk = p.chunk[0];
  A.rows_all = rows;
  A.part0 = p.parts[0] > 1 ? part : nullptr;
  if (a->dq) {
    rc = bwd_dispatch<T, false>(A, p.dc, p.parts[0], st);
    if (rc) return rc;
    if (A.part0) rc = sum_parts<T>(part, p.parts[0], rows, a->dq, Hq, Tq, D, a->dq_strides, st);
  }
  if (rc || !a->dk || a->k_len == 0) return rc;

  A.tiles = p.tiles[1];
  A.chunk = p.chunk[1];
  A.rows_all = keys;
  A.part0 = p.parts[1] > 1 ? part : nullptr;
  A.part1 = p.parts[1] > 1 ? part + p.parts[1] * keys * D : nullptr;
  rc = bwd_dispatch<T, true>(A, p.dc, p.parts[1], st);
  if (rc || !A.part0) return rc;
  rc = sum_parts<T>(A.part0, p.parts[1], keys, a->dk, Hkv, (int)a->k_len, D, a->dk_strides, st);
  if (rc) return rc;
  return sum_parts<T>(A.part1, p.parts[1], keys, a->dv, Hkv, (int)a->k_len, D, a->dv_strides, st);
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
  return a->dtype == TRNSPARSE_F32 ? bwd_simt<float>(a, ws, st) : bwd_simt<__nv_bfloat16>(a, ws, st);
}
