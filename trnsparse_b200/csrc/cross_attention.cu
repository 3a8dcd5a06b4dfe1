// Dense attention in fp32: cross attention (query rows against another
// sequence's keys, shared key heads, ragged or masked keys) and shared-prefix
// attention (decoding over one prefix for the whole batch plus each sequence's
// own keys), at any head_dim up to 256; and the bf16 shapes the tcgen05 kernels
// do not take.
//
//   s = scale q.k over the kept keys,  P = softmax(s),  O = P V
// in one pass over the keys with the running row maximum m and sum l; a row
// without keys is zero. Hidden keys never enter the arithmetic: their K and V
// rows are loaded as zeros and their scores are set to -inf, so what the
// padding holds (infinities, NaN) does not matter.
//
// Two forms. Up to 32 packed rows (decoding) are bound by the reads of K and V:
// 16 rows a CTA on the CUDA cores, a thread forming a 2 x 4 tile of scores and a
// 2 x 4 DC tile of the output from float4 reads of shared memory (32 x 16 heads, 1500
// keys of 64: 175 us, 35% of a copy's rate; 8 x 32/8 heads, up to 8192 keys of 128:
// 177 us, 24%). More rows are
// bound by arithmetic: 128 rows a CTA on the tensor cores (3xTF32, xattn_tf32.cuh),
// 48 TFLOP/s at 2 x 16/16 heads, 1024 x 1024 x 64 (180 us; 308 on the CUDA cores)
// and 50 with 16/4 heads at head_dim 128 (345 us; 615). The tensor pipe is then half
// busy: two warps a scheduler, a quarter of whose instructions are the products. bf16
// operands go the same way, though their low parts are zero (2 x 16/4 heads, 1024 x 1024:
// 970 us at head_dim 192, 1000 at 256).
// In both the next tile is copied asynchronously. When there are fewer CTAs than
// fill the GPU the keys are cut into ranges, each writing (O, log-sum-exp) of its
// part, joined afterwards.
#include <math.h>

#include "xattn_tf32.cuh"

namespace tsb {
namespace {

constexpr int kXKeys = 64;    // keys a tile: 16-row form
constexpr int kMmaKeys = 32;  // and 128-row form
// Keys of a range at most: terms are added to a range's sums in fp32, where equal ones are lost from 2^24 on.
constexpr int64_t kMostKeys = 1 << 20;

__device__ __forceinline__ float xcvt(float v) { return v; }
__device__ __forceinline__ float xcvt(__nv_bfloat16 v) { return __bfloat162float(v); }

// Four consecutive elements d .. d+3 of a D-wide row (zeros past D); vec: the row is 4-element aligned.
template <typename T>
__device__ __forceinline__ float4 load4(const T* row, int d, int D, bool vec) {
  if (vec && d + 3 < D) {
    if constexpr (sizeof(T) == 4) return *reinterpret_cast<const float4*>(row + d);
    const uint2 w = *reinterpret_cast<const uint2*>(row + d);
    return make_float4(__uint_as_float(w.x << 16), __uint_as_float(w.x & 0xffff0000u), __uint_as_float(w.y << 16),
                       __uint_as_float(w.y & 0xffff0000u));
  }
  float4 r = make_float4(0.f, 0.f, 0.f, 0.f);
  if (d < D) r.x = xcvt(row[d]);
  if (d + 1 < D) r.y = xcvt(row[d + 1]);
  if (d + 2 < D) r.z = xcvt(row[d + 2]);
  if (d + 3 < D) r.w = xcvt(row[d + 3]);
  return r;
}

template <typename T>
__device__ __forceinline__ void store1(T* p, float v) {
  if constexpr (sizeof(T) == 4) *p = v;
  else *p = __float2bfloat16_rn(v);
}

__device__ __forceinline__ float dot4(float4 a, float4 b, float c) {
  return fmaf(a.x, b.x, fmaf(a.y, b.y, fmaf(a.z, b.z, fmaf(a.w, b.w, c))));
}
__device__ __forceinline__ void fma4(float4& c, float a, float4 b) {
  c.x = fmaf(a, b.x, c.x);
  c.y = fmaf(a, b.y, c.y);
  c.z = fmaf(a, b.z, c.z);
  c.w = fmaf(a, b.w, c.w);
}

struct XKernel {
  XSide s;
  void* out;
  float *lse, *part_o, *part_lse;  // part_*: this side's first piece (null: one piece, written to out)
  int64_t rows_all;                // rows of one piece
  int D, row_tiles, chunk, vec;
  float scale_log2;
};

template <typename T, int BM, int NT, int DC>
__global__ void __launch_bounds__(NT) xattn_few_kernel(const XKernel A) {
  constexpr int TY = NT / 16, RM = BM / TY, DP = DC * 64 + 4, PP = kXKeys + 4;
  extern __shared__ __align__(16) float smx[];
  float* Qs = smx;
  float* Ks = Qs + BM * DP;
  float* Vs = Ks + kXKeys * DP;
  float* Ps = Vs + kXKeys * DP;
  const XSide& s = A.s;
  const int tid = threadIdx.x, tx = tid & 15, ty = tid >> 4;
  const int item = blockIdx.x / A.row_tiles, rt = blockIdx.x - item * A.row_tiles;
  const int bi = item / s.hkv, h = item - bi * s.hkv;
  const int64_t R = side_rows(s), r0 = static_cast<int64_t>(rt) * BM;
  const int D = A.D, len = side_len(s, bi);
  const int kbeg = blockIdx.y * A.chunk, kend = min(len, kbeg + A.chunk);
  const T* kp = static_cast<const T*>(s.k) + bi * s.k_b + h * s.k_h;
  const T* vp = static_cast<const T*>(s.v) + bi * s.v_b + h * s.v_h;
  const uint8_t* mask = s.mask ? s.mask + bi * s.mask_stride : nullptr;
  const bool vec = A.vec;
  grid_dep_launch();  // the other side's launch, which needs none of this one's results, may run beside it

  for (int i = tid; i < BM * DC * 16; i += NT) {
    const int row = i / (DC * 16), d = (i - row * (DC * 16)) * 4;
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
    if (r0 + row < R) v = load4(static_cast<const T*>(s.q) + q_offset(s, bi, h, side_row(s, r0 + row)), d, D, vec);
    *reinterpret_cast<float4*>(Qs + row * DP + d) = v;
  }
  int lim[RM];
#pragma unroll
  for (int i = 0; i < RM; ++i) {
    const int64_t r = r0 + ty * RM + i;
    lim[i] = r < R ? min(kend, row_limit(s, side_row(s, r), len)) : 0;
  }
  float m[RM], l[RM];
  float4 acc[RM][DC];
#pragma unroll
  for (int i = 0; i < RM; ++i) {
    m[i] = -INFINITY;
    l[i] = 0.f;
#pragma unroll
    for (int c = 0; c < DC; ++c) acc[i][c] = make_float4(0.f, 0.f, 0.f, 0.f);
  }
  // fp32 rows that start on 16 bytes are copied asynchronously, the others through registers
  const bool async = sizeof(T) == 4 && vec && D % 4 == 0;
  auto load_tile = [&](float* dst, const T* base, int64_t stride, int k0) {
    for (int i = tid; i < kXKeys * DC * 16; i += NT) {
      const int row = i / (DC * 16), d = (i - row * (DC * 16)) * 4;
      const int key = k0 + row;
      const bool in = key < kend && (!mask || mask[key]);
      if (async) {
        cp_async16(dst + row * DP + d, in && d < D ? base + key * stride + d : base, in && d < D);
      } else {
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
        if (in) v = load4(base + key * stride, d, D, vec);
        *reinterpret_cast<float4*>(dst + row * DP + d) = v;
      }
    }
  };
  // K of the next tile arrives while P V runs, V while the scores are formed
  if (kbeg < kend) load_tile(Ks, kp, s.k_t, kbeg);
  for (int k0 = kbeg; k0 < kend; k0 += kXKeys) {
    cp_async_wait_all();
    __syncthreads();
    load_tile(Vs, vp, s.v_t, k0);
    float sc[RM][4];
#pragma unroll
    for (int i = 0; i < RM; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) sc[i][j] = 0.f;
#pragma unroll 4
    for (int d = 0; d < DC * 64; d += 4) {
      float4 kv[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) kv[j] = *reinterpret_cast<const float4*>(Ks + (tx + 16 * j) * DP + d);
#pragma unroll
      for (int i = 0; i < RM; ++i) {
        const float4 q = *reinterpret_cast<const float4*>(Qs + (ty * RM + i) * DP + d);
#pragma unroll
        for (int j = 0; j < 4; ++j) sc[i][j] = dot4(q, kv[j], sc[i][j]);
      }
    }
    bool hid[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int key = k0 + tx + 16 * j;
      hid[j] = key >= kend || (mask && !mask[key]);
    }
#pragma unroll
    for (int i = 0; i < RM; ++i) {
      float mx = -INFINITY;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const bool hide = hid[j] || k0 + tx + 16 * j >= lim[i];
        sc[i][j] = hide ? -INFINITY : sc[i][j] * A.scale_log2;
        mx = fmaxf(mx, sc[i][j]);
      }
#pragma unroll
      for (int o = 8; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
      const float mn = fmaxf(m[i], mx);
      const float mu = mn == -INFINITY ? 0.f : mn;  // no key so far: every term is exactly 0
      const float corr = exp2f(m[i] - mu);
      float sum = 0.f;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float p = exp2f(sc[i][j] - mu);
        sum += p;
        Ps[(ty * RM + i) * PP + tx + 16 * j] = p;
      }
#pragma unroll
      for (int o = 8; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      l[i] = l[i] * corr + sum;
      m[i] = mn;
#pragma unroll
      for (int c = 0; c < DC; ++c) {
        acc[i][c].x *= corr;
        acc[i][c].y *= corr;
        acc[i][c].z *= corr;
        acc[i][c].w *= corr;
      }
    }
    cp_async_wait_all();
    __syncthreads();
    if (k0 + kXKeys < kend) load_tile(Ks, kp, s.k_t, k0 + kXKeys);
#pragma unroll 2
    for (int k = 0; k < kXKeys; k += 4) {
      float4 p[RM];
#pragma unroll
      for (int i = 0; i < RM; ++i) p[i] = *reinterpret_cast<const float4*>(Ps + (ty * RM + i) * PP + k);
#pragma unroll
      for (int kk = 0; kk < 4; ++kk)
#pragma unroll
        for (int c = 0; c < DC; ++c) {
          const float4 v = *reinterpret_cast<const float4*>(Vs + (k + kk) * DP + tx * 4 + 64 * c);
#pragma unroll
          for (int i = 0; i < RM; ++i)
            fma4(acc[i][c], kk == 0 ? p[i].x : kk == 1 ? p[i].y : kk == 2 ? p[i].z : p[i].w, v);
        }
    }
  }
#pragma unroll
  for (int i = 0; i < RM; ++i) {
    const int64_t r = r0 + ty * RM + i;
    if (r >= R) continue;
    const XRow x = side_row(s, r);
    const int64_t fr = flat_row(s, bi, h, x);
    const float inv = l[i] > 0.f ? 1.f / l[i] : (l[i] == 0.f ? 0.f : l[i]);
    const float lse = l[i] == 0.f ? -INFINITY : m[i] + log2f(l[i]);
    if (A.part_o != nullptr) {
      float* po = A.part_o + (static_cast<int64_t>(blockIdx.y) * A.rows_all + fr) * D;
      for (int c = 0; c < DC; ++c) {
        const int d = tx * 4 + 64 * c;
        const float e[4] = {acc[i][c].x, acc[i][c].y, acc[i][c].z, acc[i][c].w};
#pragma unroll
        for (int q = 0; q < 4; ++q)
          if (d + q < D) po[d + q] = e[q] * inv;
      }
      if (tx == 0) A.part_lse[static_cast<int64_t>(blockIdx.y) * A.rows_all + fr] = lse;
    } else {
      T* po = static_cast<T*>(A.out) + o_offset(s, bi, h, x);
      for (int c = 0; c < DC; ++c) {
        const int d = tx * 4 + 64 * c;
        const float e[4] = {acc[i][c].x, acc[i][c].y, acc[i][c].z, acc[i][c].w};
#pragma unroll
        for (int q = 0; q < 4; ++q)
          if (d + q < D) store1(po + d + q, e[q] * inv);
      }
      if (A.lse != nullptr && tx == 0) A.lse[fr] = lse;
    }
  }
  grid_dep_wait();  // ends after the launch it ran beside: what follows needs both
}

// 128 rows a CTA: four warps of 32, so that each split of a K or V element feeds two products, or (above head_dim 128,
// where 32 rows' sums would not fit in registers) eight of 16. Scores and probabilities stay in registers.
template <typename T, int DC>
__global__ void __launch_bounds__(DC == 4 ? 256 : 128, DC <= 2 ? 2 : 1) xattn_mma_kernel(const XKernel A) {
  constexpr int BM = 128, MT = DC == 4 ? 1 : 2, NT = DC == 4 ? 256 : 128, KT = kMmaKeys;
  constexpr int DP = DC * 64 + 4, NK = KT / 8, NO = DC * 8, CH = DC * 16;
  extern __shared__ __align__(16) float smx[];
  float* Qs = smx;
  float* Ks = Qs + BM * DP;
  float* Vs = Ks + KT * DP;
  const XSide& s = A.s;
  const int tid = threadIdx.x, lane = tid & 31, wr = (tid >> 5) * 16 * MT, g = lane >> 2, t = lane & 3;
  const int item = blockIdx.x / A.row_tiles, rt = blockIdx.x - item * A.row_tiles;
  const int bi = item / s.hkv, h = item - bi * s.hkv;
  const int64_t R = side_rows(s), r0 = static_cast<int64_t>(rt) * BM;
  const int D = A.D, len = side_len(s, bi);
  const int kbeg = blockIdx.y * A.chunk, kend = min(len, kbeg + A.chunk);
  const T* kp = static_cast<const T*>(s.k) + bi * s.k_b + h * s.k_h;
  const T* vp = static_cast<const T*>(s.v) + bi * s.v_b + h * s.v_h;
  const uint8_t* mask = s.mask ? s.mask + bi * s.mask_stride : nullptr;
  const bool busy = r0 + wr < R;  // a warp without rows only copies
  grid_dep_launch();  // the other side's launch, which needs none of this one's results, may run beside it

  for (int i = tid; i < BM * CH; i += NT) {
    const int row = i / CH, d = (i - row * CH) * 4;
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
    if (r0 + row < R) v = load4(static_cast<const T*>(s.q) + q_offset(s, bi, h, side_row(s, r0 + row)), d, D, A.vec);
    *reinterpret_cast<float4*>(Qs + row * DP + d) = v;
  }
  int lim[MT][2], least = kend;
  float m[MT][2], l[MT][2], acc[MT][NO][4];
#pragma unroll
  for (int a = 0; a < MT; ++a) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int64_t r = r0 + wr + a * 16 + g + 8 * i;
      lim[a][i] = r < R ? min(kend, row_limit(s, side_row(s, r), len)) : kend;
      least = min(least, lim[a][i]);
      m[a][i] = -INFINITY;
      l[a][i] = 0.f;
    }
#pragma unroll
    for (int n = 0; n < NO; ++n)
#pragma unroll
      for (int j = 0; j < 4; ++j) acc[a][n][j] = 0.f;
  }
  // fp32 rows that start on 16 bytes are copied asynchronously, the others through registers
  const bool async = sizeof(T) == 4 && A.vec && D % 4 == 0;
  const int c_row = tid / CH, c_d = (tid % CH) * 4;  // this thread's first row and its columns
  auto load_tile = [&](float* dst, const T* base, int64_t stride, int k0) {
    if (async) {
      const T* src = base + (k0 + c_row) * stride + c_d;
      const bool any = c_d < D;
#pragma unroll 4
      for (int row = c_row; row < KT; row += NT / CH, src += NT / CH * stride) {
        const bool in = any && k0 + row < kend && (!mask || mask[k0 + row]);
        cp_async16(dst + row * DP + c_d, in ? src : base, in);
      }
    } else {
      for (int row = c_row; row < KT; row += NT / CH) {
        const int key = k0 + row;
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
        if (key < kend && (!mask || mask[key])) v = load4(base + key * stride, c_d, D, A.vec);
        *reinterpret_cast<float4*>(dst + row * DP + c_d) = v;
      }
    }
  };
  // K of the next tile arrives while P V runs, V while the scores are formed
  if (kbeg < kend) load_tile(Ks, kp, s.k_t, kbeg);
  for (int k0 = kbeg; k0 < kend; k0 += KT) {
    cp_async_wait_all();
    __syncthreads();
    load_tile(Vs, vp, s.v_t, k0);
    float sc[MT][NK][4];
    if (busy) {
#pragma unroll
      for (int a = 0; a < MT; ++a)
#pragma unroll
        for (int n = 0; n < NK; ++n)
#pragma unroll
          for (int j = 0; j < 4; ++j) sc[a][n][j] = 0.f;
      static_assert(KT == 32, "a lane a key");
      const bool check = mask || k0 + KT > least;
      bool seen = true;  // key k0 + lane
      if (check) seen = k0 + lane < kend && (!mask || mask[k0 + lane]);
      scores_tf32<MT, NK, DP>(sc, Qs + wr * DP, Ks, D, g, t);
#pragma unroll
      for (int a = 0; a < MT; ++a)
#pragma unroll
        for (int n = 0; n < NK; ++n)
#pragma unroll
          for (int j = 0; j < 4; ++j) sc[a][n][j] *= A.scale_log2;
      if (__any_sync(0xffffffffu, check)) {
        const unsigned keep = __ballot_sync(0xffffffffu, seen);
#pragma unroll
        for (int n = 0; n < NK; ++n)
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const int x = n * 8 + 2 * t + j, key = k0 + x;
            const bool hid = !(keep >> x & 1u);
#pragma unroll
            for (int a = 0; a < MT; ++a)
#pragma unroll
              for (int i = 0; i < 2; ++i)
                if (hid || key >= lim[a][i]) sc[a][n][2 * i + j] = -INFINITY;
          }
      }
#pragma unroll
      for (int a = 0; a < MT; ++a)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          float mx = -INFINITY;
#pragma unroll
          for (int n = 0; n < NK; ++n) mx = fmaxf(mx, fmaxf(sc[a][n][2 * i], sc[a][n][2 * i + 1]));
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
          const float mn = fmaxf(m[a][i], mx);
          const float mu = mn == -INFINITY ? 0.f : mn;  // no key so far: every term is exactly 0
          const float corr = ex2(m[a][i] - mu);
          m[a][i] = mn;
          float sum = 0.f;
#pragma unroll
          for (int n = 0; n < NK; ++n)
#pragma unroll
            for (int j = 2 * i; j < 2 * i + 2; ++j) {
              sc[a][n][j] = ex2(sc[a][n][j] - mu);
              sum += sc[a][n][j];
            }
          l[a][i] = l[a][i] * corr + sum;  // this lane's columns; the four lanes' sums are joined at the end
#pragma unroll
          for (int n = 0; n < NO; ++n) {
            acc[a][n][2 * i] *= corr;
            acc[a][n][2 * i + 1] *= corr;
          }
        }
    }
    cp_async_wait_all();
    __syncthreads();
    if (k0 + KT < kend) load_tile(Ks, kp, s.k_t, k0 + KT);
    if (busy) weigh_tf32<MT, NK, NO, DP>(acc, sc, Vs, g, t);
  }
#pragma unroll
  for (int a = 0; a < MT; ++a)
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      float ls = l[a][i];
      ls += __shfl_xor_sync(0xffffffffu, ls, 1);
      ls += __shfl_xor_sync(0xffffffffu, ls, 2);
      const int64_t r = r0 + wr + a * 16 + g + 8 * i;
      if (r >= R) continue;
      const XRow x = side_row(s, r);
      const int64_t fr = flat_row(s, bi, h, x);
      const float inv = ls > 0.f ? 1.f / ls : (ls == 0.f ? 0.f : ls);
      const float lse = ls == 0.f ? -INFINITY : m[a][i] + log2f(ls);
      const bool piece = A.part_o != nullptr;
      const int64_t pr = static_cast<int64_t>(blockIdx.y) * A.rows_all + fr;
      float* pp = piece ? A.part_o + pr * D : nullptr;
      T* po = piece ? nullptr : static_cast<T*>(A.out) + o_offset(s, bi, h, x);
#pragma unroll
      for (int n = 0; n < NO; ++n)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const int d = n * 8 + 2 * t + j;
          const float v = acc[a][n][2 * i + j] * inv;
          if (d < D) {
            if (piece) pp[d] = v;
            else store1(po + d, v);
          }
        }
      if (t == 0) {
        if (piece) A.part_lse[pr] = lse;
        else if (A.lse != nullptr) A.lse[fr] = lse;
      }
    }
  grid_dep_wait();  // ends after the launch it ran beside: what follows needs both
}

// One warp per row.
template <typename T>
__global__ void __launch_bounds__(256) combine_pieces_kernel(const float* __restrict__ part_o,
                                                             const float* __restrict__ part_lse, int pieces,
                                                             int64_t rows, T* out, float* lse, int64_t o_b,
                                                             int64_t o_h, int64_t o_t, int Hq, int Tq, int D) {
  const int64_t row = static_cast<int64_t>(blockIdx.x) * 8 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  if (row >= rows) return;
  float mx = -INFINITY;
  for (int p = lane; p < pieces; p += 32) mx = fmaxf(mx, part_lse[p * rows + row]);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
  const float mu = mx == -INFINITY ? 0.f : mx;
  float acc[8], den = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) acc[i] = 0.f;
  // four pieces' loads in flight together
  for (int p0 = 0; p0 < pieces; p0 += 4) {
    float lp[4], v[4][8];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const bool in = p0 + k < pieces;
      lp[k] = in ? part_lse[(p0 + k) * rows + row] : -INFINITY;
      const float* po = part_o + ((p0 + k) * rows + row) * D;
#pragma unroll
      for (int i = 0; i < 8; ++i) v[k][i] = in && lane + 32 * i < D ? po[lane + 32 * i] : 0.f;
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float w = exp2f(lp[k] - mu);  // an empty piece holds zeros and weighs 0
      den += w;
#pragma unroll
      for (int i = 0; i < 8; ++i) acc[i] = fmaf(w, v[k][i], acc[i]);
    }
  }
  const int t = static_cast<int>(row % Tq);
  const int64_t bh = row / Tq, b = bh / Hq, h = bh - b * Hq;
  T* po = out + b * o_b + h * o_h + t * o_t;
  const float inv = den == 0.f ? 0.f : 1.f / den;
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (lane + 32 * i < D) store1(po + lane + 32 * i, acc[i] * inv);
  if (lse != nullptr && lane == 0) lse[row] = den == 0.f ? -INFINITY : mx + log2f(den);
}

// ---------------------------------------------------------------- host side

struct GeneralPlan {
  int dc, bm[2], splits[2], chunk[2], row_tiles[2], pieces;
};

GeneralPlan general_plan(const trnsparse_attention_args* a, const XSide (&s)[2], int n) {
  GeneralPlan p = {};
  p.dc = a->head_dim <= 64 ? 1 : a->head_dim <= 128 ? 2 : 4;
  const int resident = p.dc <= 2 ? 2 : 1;  // CTAs an SM: by registers and shared memory
  for (int i = 0; i < n; ++i) {
    p.bm[i] = side_rows(s[i]) <= 32 ? 16 : 128;  // 16-row CTAs where a 128-row tile would be mostly padding
    const int64_t keys = p.bm[i] == 16 ? kXKeys : kMmaKeys;
    p.row_tiles[i] = static_cast<int>((side_rows(s[i]) + p.bm[i] - 1) / p.bm[i]);
    const int64_t ctas = static_cast<int64_t>(p.row_tiles[i]) * s[i].nb * s[i].hkv;
    const int64_t tiles = (s[i].klen + keys - 1) / keys;
    int64_t per;
    // bound by the reads of K and V: three CTAs an SM (walk_steps' fewer: 46 us against 31 at 4096 keys)
    if (p.bm[i] == 16) {
      int64_t splits = ctas > 0 ? (3ll * sm_count() + ctas - 1) / ctas : 1;
      splits = splits < 128 ? splits : 128;
      per = tiles > splits ? (tiles + splits - 1) / splits : 1;
    } else {
      per = walk_steps(ctas, tiles, sm_count(), resident, 128, 0.1);
    }
    if (per > kMostKeys / keys) per = kMostKeys / keys;
    p.chunk[i] = static_cast<int>(per * keys);
    p.splits[i] = static_cast<int>(tiles > 0 ? (tiles + per - 1) / per : 1);
    p.pieces += p.splits[i];
  }
  return p;
}

int attention_launch(void (*kern)(XKernel), int threads, size_t smem, const XKernel& A, int splits, bool behind,
                     cudaStream_t st) {
  cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem));
  if (e != cudaSuccess) return cuda_status(e, "attention: set smem");
  const dim3 grid(static_cast<unsigned>(A.row_tiles) * A.s.nb * A.s.hkv, splits);
  if (behind) {
    e = launch_pdl(kern, grid, dim3(threads), smem, st, A);
    return e == cudaSuccess ? TRNSPARSE_OK : cuda_status(e, "attention launch");
  }
  kern<<<grid, threads, smem, st>>>(A);
  TSB_CHECK_LAUNCH("attention launch");
  return TRNSPARSE_OK;
}

template <typename T, int DC>
int attention_dispatch(const XKernel& A, int bm, int splits, bool behind, cudaStream_t st) {
  const size_t row = sizeof(float) * (DC * 64 + 4);
  if (bm == 128)
    return attention_launch(xattn_mma_kernel<T, DC>, DC == 4 ? 256 : 128, row * (128 + 2 * kMmaKeys), A, splits, behind,
                            st);
  return attention_launch(xattn_few_kernel<T, 16, 128, DC>, 128,
                          row * (16 + 2 * kXKeys) + sizeof(float) * 16 * (kXKeys + 4), A, splits, behind, st);
}

template <typename T>
int general_dispatch(const XKernel& A, int bm, int dc, int splits, bool behind, cudaStream_t st) {
  if (dc == 1) return attention_dispatch<T, 1>(A, bm, splits, behind, st);
  if (dc == 2) return attention_dispatch<T, 2>(A, bm, splits, behind, st);
  return attention_dispatch<T, 4>(A, bm, splits, behind, st);
}

// Every base and stride of the call's operands is a multiple of four elements.
bool four_aligned(const trnsparse_attention_args* a) {
  const uintptr_t m = a->dtype == TRNSPARSE_F32 ? 15 : 7;
  uintptr_t p = reinterpret_cast<uintptr_t>(a->q) | reinterpret_cast<uintptr_t>(a->k) |
                reinterpret_cast<uintptr_t>(a->v) | reinterpret_cast<uintptr_t>(a->prefix_k) |
                reinterpret_cast<uintptr_t>(a->prefix_v);
  int64_t st = 0;
  for (int i = 0; i < 3; ++i) st |= a->q_strides[i] | a->k_strides[i] | a->v_strides[i];
  for (int i = 0; i < 2; ++i) st |= a->prefix_k_strides[i] | a->prefix_v_strides[i];
  return !(p & m) && !(st & 3);
}

int general_forward(const trnsparse_attention_args* a, bool prefix, void* ws, cudaStream_t st) {
  XSide s[2];
  int n = 0;
  int rc = make_sides(a, prefix, s, &n);
  if (rc) return rc;
  const GeneralPlan p = general_plan(a, s, n);
  const int64_t rows = a->batch * a->q_heads * a->q_len;
  float* part_o = static_cast<float*>(ws);
  float* part_lse = part_o + (p.pieces > 1 ? p.pieces * rows * a->head_dim : 0);
  int piece = 0;
  for (int i = 0; i < n; ++i) {
    XKernel A = {};
    A.s = s[i];
    A.out = a->out;
    A.lse = a->lse;
    if (p.pieces > 1) {
      A.part_o = part_o + piece * rows * a->head_dim;
      A.part_lse = part_lse + piece * rows;
    }
    A.rows_all = rows;
    A.D = static_cast<int>(a->head_dim);
    A.row_tiles = p.row_tiles[i];
    A.chunk = p.chunk[i];
    A.vec = four_aligned(a);
    A.scale_log2 = static_cast<float>(a->scale * 1.4426950408889634);
    rc = a->dtype == TRNSPARSE_F32 ? general_dispatch<float>(A, p.bm[i], p.dc, p.splits[i], i > 0, st)
                                   : general_dispatch<__nv_bfloat16>(A, p.bm[i], p.dc, p.splits[i], i > 0, st);
    if (rc) return rc;
    piece += p.splits[i];
  }
  return p.pieces > 1 ? combine_pieces(part_o, part_lse, p.pieces, a, st) : TRNSPARSE_OK;
}

size_t general_workspace(const trnsparse_attention_args* a, bool prefix) {
  XSide s[2];
  int n = 0;
  if (make_sides(a, prefix, s, &n)) return 0;
  const GeneralPlan p = general_plan(a, s, n);
  if (p.pieces <= 1) return 0;
  return sizeof(float) * static_cast<size_t>(p.pieces) * a->batch * a->q_heads * a->q_len * (a->head_dim + 1);
}

}  // namespace

int combine_pieces(const float* part_o, const float* part_lse, int pieces, const trnsparse_attention_args* a,
                   cudaStream_t st) {
  const int64_t rows = a->batch * a->q_heads * a->q_len;
  const unsigned grid = static_cast<unsigned>((rows + 7) / 8);
  const int64_t* os = a->out_strides;
  if (a->dtype == TRNSPARSE_F32)
    combine_pieces_kernel<float><<<grid, 256, 0, st>>>(part_o, part_lse, pieces, rows, static_cast<float*>(a->out),
                                                       a->lse, os[0], os[1], os[2], (int)a->q_heads, (int)a->q_len,
                                                       (int)a->head_dim);
  else
    combine_pieces_kernel<__nv_bfloat16><<<grid, 256, 0, st>>>(
        part_o, part_lse, pieces, rows, static_cast<__nv_bfloat16*>(a->out), a->lse, os[0], os[1], os[2],
        (int)a->q_heads, (int)a->q_len, (int)a->head_dim);
  TSB_CHECK_LAUNCH("attention combine launch");
  return TRNSPARSE_OK;
}

int check_attention(const trnsparse_attention_args* a, const char* what) {
  TSB_REQUIRE(a != nullptr, "%s: null arguments", what);
  TSB_REQUIRE(a->batch >= 0 && a->q_heads >= 0 && a->kv_heads >= 0 && a->q_len >= 0 && a->k_len >= 0 &&
                  a->prefix_len >= 0,
              "%s: negative size", what);
  TSB_REQUIRE(a->head_dim >= 1 && a->head_dim <= 256, "%s: head_dim must be in [1, 256] (got %lld)", what,
              (long long)a->head_dim);
  TSB_REQUIRE(a->q_heads == 0 || (a->kv_heads > 0 && a->q_heads % a->kv_heads == 0),
              "%s: %lld query heads are not a multiple of %lld key heads", what, (long long)a->q_heads,
              (long long)a->kv_heads);
  TSB_REQUIRE(a->k_len < (1ll << 30) && a->prefix_len < (1ll << 30) && a->batch < (1ll << 24) &&
                  a->q_heads < (1 << 16) && a->q_len < (1ll << 30) &&
                  a->batch * a->q_heads < (1ll << 30) && a->batch * a->q_heads * a->q_len < (1ll << 30),
              "%s: sizes out of range", what);
  // the kernels scale by this in fp32; a NaN would pass the tensor cores' lower bound on it as if it were 0
  TSB_REQUIRE(isfinite(static_cast<float>(a->scale * 1.4426950408889634)), "%s: scale %g is not finite in fp32", what,
              a->scale);
  if (a->dtype != TRNSPARSE_F32 && a->dtype != TRNSPARSE_BF16)
    return fail(TRNSPARSE_ERR_DTYPE, "%s: dtype %d not supported (F32, BF16)", what, a->dtype);
  return TRNSPARSE_OK;
}

int make_sides(const trnsparse_attention_args* a, bool prefix, XSide (&s)[2], int* n) {
  XSide c = {};
  c.q = a->q;
  c.q_h = a->q_strides[1];
  c.q_t = a->q_strides[2];
  c.o_h = a->out_strides[1];
  c.o_t = a->out_strides[2];
  c.hkv = static_cast<int>(a->kv_heads);
  c.G = static_cast<int>(a->q_heads / a->kv_heads);
  c.T = static_cast<int>(a->q_len);
  *n = 0;
  if (prefix && a->prefix_len > 0) {
    XSide& p = s[(*n)++];
    p = c;
    p.k = a->prefix_k;
    p.v = a->prefix_v;
    p.q_b2 = a->q_strides[0];
    p.o_b2 = a->out_strides[0];
    p.k_h = a->prefix_k_strides[0];
    p.k_t = a->prefix_k_strides[1];
    p.v_h = a->prefix_v_strides[0];
    p.v_t = a->prefix_v_strides[1];
    p.nb = 1;
    p.n2 = static_cast<int>(a->batch);
    p.klen = static_cast<int>(a->prefix_len);
  }
  if (a->k_len > 0 || *n == 0) {
    XSide& o = s[(*n)++];
    o = c;
    o.k = a->k;
    o.v = a->v;
    o.q_bi = a->q_strides[0];
    o.o_bi = a->out_strides[0];
    o.k_b = a->k_strides[0];
    o.k_h = a->k_strides[1];
    o.k_t = a->k_strides[2];
    o.v_b = a->v_strides[0];
    o.v_h = a->v_strides[1];
    o.v_t = a->v_strides[2];
    o.lengths = a->key_lengths;
    o.mask = a->key_mask;
    o.mask_stride = a->key_mask_stride;
    o.nb = static_cast<int>(a->batch);
    o.n2 = 1;
    o.klen = static_cast<int>(a->k_len);
    o.causal = prefix ? 1 : 0;
  }
  return TRNSPARSE_OK;
}

namespace {

bool nothing(const trnsparse_attention_args* a) { return a->batch * a->q_heads * a->q_len == 0; }

size_t attention_workspace(const trnsparse_attention_args* a, bool prefix) {
  if (check_attention(a, "attention") || nothing(a)) return 0;
  return xattn_tc_ok(a, prefix) ? xattn_tc_workspace(a, prefix) : general_workspace(a, prefix);
}

int attention_run(const trnsparse_attention_args* a, bool prefix, void* ws, size_t ws_bytes, void* stream,
                  const char* what) {
  int rc = check_attention(a, what);
  if (rc) return rc;
  if (nothing(a)) return TRNSPARSE_OK;
  TSB_REQUIRE(a->q && a->out && (a->k_len == 0 || (a->k && a->v)) &&
                  (!prefix || a->prefix_len == 0 || (a->prefix_k && a->prefix_v)),
              "%s: null pointer", what);
  const size_t need = attention_workspace(a, prefix);
  TSB_REQUIRE(ws_bytes >= need && (need == 0 || ws), "%s: workspace too small (%zu bytes, needs %zu)", what, ws_bytes,
              need);
  return xattn_tc_ok(a, prefix) ? xattn_tc_forward(a, prefix, ws, as_stream(stream))
                                : general_forward(a, prefix, ws, as_stream(stream));
}

}  // namespace
}  // namespace tsb

using namespace tsb;

extern "C" size_t trnsparse_cross_attention_workspace_size(const trnsparse_attention_args* args) {
  return attention_workspace(args, false);
}
extern "C" int trnsparse_cross_attention(const trnsparse_attention_args* args, void* ws, size_t ws_bytes,
                                         void* stream) {
  return attention_run(args, false, ws, ws_bytes, stream, "cross_attention");
}
extern "C" size_t trnsparse_shared_prefix_attention_workspace_size(const trnsparse_attention_args* args) {
  return attention_workspace(args, true);
}
extern "C" int trnsparse_shared_prefix_attention(const trnsparse_attention_args* args, void* ws, size_t ws_bytes,
                                                 void* stream) {
  return attention_run(args, true, ws, ws_bytes, stream, "shared_prefix_attention");
}
