// RMS norm of every query and key head with the position rotation in the same
// pass, forward and backward. For a head vector x (D wide), r = (mean x_i^2 +
// eps)^(-1/2), n_i = x_i r w_i, and the pair (a, b) number j of the first R
// elements is turned by the angle p f_j of the token's position p:
//   y_a = n_a cos - n_b sin,  y_b = n_b cos + n_a sin
// (pair j = (j, j + R/2), or (2j, 2j + 1) when interleaved; elements past R
// pass). Backward, with u = x r and Rot^T the turn the other way:
//   dn = Rot^T dy,  dw = sum over rows of dn u,  g = dn w,
//   dx = r (g - u mean(g u)).
//
// What bounds it: memory; x is read and y written once (backward: x, dy read,
// dx written). The one costly scalar part is the angle: p f_j in 64 bits (a
// 32-bit product is off by a radian near p = 10^7), taken modulo a full turn in
// 64 bits and only then rounded, by 2^-26 of a turn at most: an angle is off by up to
// 9.4e-8 at any position, less than a step of fp32. It
// depends on the token and the pair alone, so a group of lanes owns one token,
// keeps its cosines and sines in registers and walks over the token's heads.
// Lane l of a group holds unit l: VEC elements from each side of VEC pairs, so
// a rotation needs no exchange between lanes and every access is one vector.
// Sums of squares and all products are fp32; y and dx are rounded once.
// dw: each thread adds its rows' terms in fp32 registers, a CTA joins its
// groups in shared memory into one partial row, and a second launch adds the
// partial rows in a fixed order (no atomics: results repeat bit for bit).
// 16384 tokens of 2 x 16 bf16 heads of 128: forward and backward 144 us of kernels for
// 671 MB, 4.7 TB/s, 72% of a copy's rate.
#include <cuda_bf16.h>

#include "common.cuh"

namespace tsb {
namespace {

constexpr int kQkThreads = 256;

struct QkTensor {
  const void* x;
  const void* dy;
  void* out;  // y forward, dx backward
  const void* w;
  float* dw_part;
  int64_t xs[3], dys[3], os[3];  // strides (batch, head, token) in elements
  int heads, chunks;
};

struct QkArgs {
  QkTensor t[2];
  const void* pos;
  const double* freq;
  int64_t tokens, pos_stride;  // tokens = B * S; pos_stride: 0 (one row for the batch) or S's stride
  int S, D, R, pos64, w_bf16, head_chunk;
  float eps, inv_d;
};

// VEC elements as they lie in memory, and as floats.
template <typename T, int VEC>
struct Raw {
  uint32_t w[VEC == 1 ? 1 : VEC * sizeof(T) / 4];
};
template <typename T, int VEC>
__device__ __forceinline__ void load_raw(const T* p, Raw<T, VEC>& v) {
  if constexpr (VEC == 1 && sizeof(T) == 2) v.w[0] = static_cast<uint32_t>(*reinterpret_cast<const uint16_t*>(p)) << 16;
  else if constexpr (VEC == 1) v.w[0] = __float_as_uint(*reinterpret_cast<const float*>(p));
  else if constexpr (sizeof(T) == 4) *reinterpret_cast<uint4*>(v.w) = *reinterpret_cast<const uint4*>(p);
  else *reinterpret_cast<uint2*>(v.w) = *reinterpret_cast<const uint2*>(p);
}
template <typename T, int VEC>
__device__ __forceinline__ void to_floats(const Raw<T, VEC>& r, float (&v)[VEC]) {
#pragma unroll
  for (int i = 0; i < VEC; ++i) {
    if constexpr (VEC == 1 || sizeof(T) == 4) v[i] = __uint_as_float(r.w[i]);
    else v[i] = __uint_as_float(i & 1 ? r.w[i / 2] & 0xffff0000u : r.w[i / 2] << 16);
  }
}

template <typename T, int VEC>
__device__ __forceinline__ void store_vec(T* p, const float (&v)[VEC]) {
  if constexpr (VEC == 1) {
    if constexpr (sizeof(T) == 4) p[0] = v[0];
    else p[0] = __float2bfloat16_rn(v[0]);
  } else if constexpr (sizeof(T) == 4) {
    *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
  } else {
    uint32_t w[VEC / 2];
#pragma unroll
    for (int i = 0; i < VEC / 2; ++i) {
      __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
      w[i] = *reinterpret_cast<uint32_t*>(&h);
    }
    *reinterpret_cast<uint2*>(p) = *reinterpret_cast<uint2*>(w);
  }
}

// The two VEC-wide pieces of a unit, as the pair sides a and b. Halves: the
// pieces are the sides. Interleaved: the pieces are 2 VEC adjacent elements.
template <int VEC, bool INTER>
__device__ __forceinline__ void to_pairs(float (&a)[VEC], float (&b)[VEC]) {
  if constexpr (INTER && VEC > 1) {
    float t[2 * VEC];
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      t[i] = a[i];
      t[VEC + i] = b[i];
    }
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      a[i] = t[2 * i];
      b[i] = t[2 * i + 1];
    }
  }
}
template <int VEC, bool INTER>
__device__ __forceinline__ void from_pairs(float (&a)[VEC], float (&b)[VEC]) {
  if constexpr (INTER && VEC > 1) {
    float t[2 * VEC];
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      t[2 * i] = a[i];
      t[2 * i + 1] = b[i];
    }
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      a[i] = t[i];
      b[i] = t[VEC + i];
    }
  }
}

// KU units per lane (VEC == 1 only: up to 128 units on 32 lanes), LPR lanes per token.
template <typename T, int VEC, int KU, bool INTER, bool BWD>
__global__ void __launch_bounds__(kQkThreads, VEC == 1 ? 1 : BWD ? 2 : 4) qk_norm_rope_kernel(const QkArgs A, int lpr) {
  extern __shared__ float sm_dw[];
  const int which = static_cast<int>(blockIdx.y) < A.t[0].chunks ? 0 : 1;
  const QkTensor& t = A.t[which];
  const int chunk = blockIdx.y - (which ? A.t[0].chunks : 0);
  const int h0 = chunk * A.head_chunk, h1 = min(h0 + A.head_chunk, t.heads);
  const int groups = kQkThreads / lpr, grp = threadIdx.x / lpr, lane = threadIdx.x % lpr;
  const int D = A.D, R = A.R;
  const int rot_units = R / (2 * VEC), units = (D + 2 * VEC - 1) / (2 * VEC);

  int o1[KU], o2[KU];  // element offsets of a unit's pieces; -1: none
  float wa[KU][VEC], wb[KU][VEC], dwa[KU][VEC], dwb[KU][VEC];
#pragma unroll
  for (int u = 0; u < KU; ++u) {
    const int unit = lane + u * lpr;
    if (unit >= units) {
      o1[u] = o2[u] = -1;
    } else if (unit < rot_units && !INTER) {
      o1[u] = unit * VEC;
      o2[u] = R / 2 + unit * VEC;
    } else {  // adjacent pieces: interleaved pairs, or elements that pass
      o1[u] = unit * 2 * VEC;
      o2[u] = o1[u] + VEC < D ? o1[u] + VEC : -1;
    }
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      wa[u][i] = wb[u][i] = 1.f;
      dwa[u][i] = dwb[u][i] = 0.f;
      if (t.w != nullptr) {
        auto wv = [&](int e) {
          return A.w_bf16 ? __bfloat162float(static_cast<const __nv_bfloat16*>(t.w)[e]) : static_cast<const float*>(t.w)[e];
        };
        if (o1[u] >= 0) wa[u][i] = wv(o1[u] + i);
        if (o2[u] >= 0) wb[u][i] = wv(o2[u] + i);
      }
    }
    to_pairs<VEC, INTER>(wa[u], wb[u]);
  }

  const int64_t step = static_cast<int64_t>(gridDim.x) * groups;
  // every lane of a warp makes the same number of steps (shuffles below); the last may be idle
  for (int64_t base = static_cast<int64_t>(blockIdx.x) * groups; base < A.tokens; base += step) {
    const int64_t tok = base + grp;
    const bool live = tok < A.tokens;
    const int64_t bi = live ? tok / A.S : 0, si = live ? tok - bi * A.S : 0;
    float cs[KU][VEC], sn[KU][VEC];
    const int64_t pi = bi * A.pos_stride + si;
    const double p = A.pos64 ? static_cast<double>(static_cast<const int64_t*>(A.pos)[pi])
                             : static_cast<double>(static_cast<const int*>(A.pos)[pi]);
#pragma unroll
    for (int u = 0; u < KU; ++u) {
      const int unit = lane + u * lpr;
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        cs[u][i] = 1.f;
        sn[u][i] = 0.f;
        if (unit < rot_units) {
          double turn = p * A.freq[unit * VEC + i] * 0.15915494309189535;  // angle / (2 pi)
          turn -= rint(turn);
          sincospif(2.f * static_cast<float>(turn), &sn[u][i], &cs[u][i]);
        }
      }
    }
    const T* xt = static_cast<const T*>(t.x) + bi * t.xs[0] + h0 * t.xs[1] + si * t.xs[2];
    const T* dyt = BWD ? static_cast<const T*>(t.dy) + bi * t.dys[0] + h0 * t.dys[1] + si * t.dys[2] : nullptr;
    T* ot = static_cast<T*>(t.out) + bi * t.os[0] + h0 * t.os[1] + si * t.os[2];
    // The next DEPTH heads' vectors are in flight while this head's are used, as many as registers allow. bf16, 16384
    // tokens of 2 x 16 heads of 128: forward 1 or 2 heads 64.4, 56.3 us; backward 1 head on three CTAs an SM or 3 on two
    // 89.8, 84.6 us.
    constexpr int DEPTH = VEC == 1 ? 1 : sizeof(T) == 2 ? (BWD ? 3 : 2) : (BWD ? 2 : 1);
    Raw<T, VEC> rx[DEPTH][KU][2], rd[DEPTH][BWD ? KU : 1][2];
    auto fetch = [&](int n) {
#pragma unroll
      for (int u = 0; u < KU; ++u)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int o = e ? o2[u] : o1[u];
          if (live && o >= 0) {
            load_raw<T, VEC>(xt + o, rx[n][u][e]);
            if constexpr (BWD) load_raw<T, VEC>(dyt + o, rd[n][u][e]);
          }
        }
      xt += t.xs[1];
      if constexpr (BWD) dyt += t.dys[1];
    };
#pragma unroll
    for (int n = 0; n < DEPTH; ++n) {
#pragma unroll
      for (int u = 0; u < KU; ++u)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          rx[n][u][e] = Raw<T, VEC>{};
          if constexpr (BWD) rd[n][u][e] = Raw<T, VEC>{};
        }
      if (h0 + n < h1) fetch(n);
    }
    for (int hb = h0; hb < h1; hb += DEPTH)
#pragma unroll
    for (int n = 0; n < DEPTH; ++n) {
      const int h = hb + n;
      if (h >= h1) break;
      float a[KU][VEC], b[KU][VEC], ga[KU][VEC], gb[KU][VEC];
      float ss = 0.f, gx = 0.f;
#pragma unroll
      for (int u = 0; u < KU; ++u) {
        to_floats<T, VEC>(rx[n][u][0], a[u]);
        to_floats<T, VEC>(rx[n][u][1], b[u]);
        if constexpr (BWD) {
          to_floats<T, VEC>(rd[n][u][0], ga[u]);
          to_floats<T, VEC>(rd[n][u][1], gb[u]);
        }
      }
      if (h + DEPTH < h1) fetch(n);
#pragma unroll
      for (int u = 0; u < KU; ++u) {
        to_pairs<VEC, INTER>(a[u], b[u]);
        if constexpr (BWD) to_pairs<VEC, INTER>(ga[u], gb[u]);
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          ss = fmaf(a[u][i], a[u][i], fmaf(b[u][i], b[u][i], ss));
          if constexpr (BWD) {
            const float da = ga[u][i], db = gb[u][i];
            ga[u][i] = fmaf(da, cs[u][i], db * sn[u][i]);
            gb[u][i] = fmaf(db, cs[u][i], -da * sn[u][i]);
            gx = fmaf(ga[u][i] * wa[u][i], a[u][i], fmaf(gb[u][i] * wb[u][i], b[u][i], gx));
          }
        }
      }
      for (int o = lpr >> 1; o > 0; o >>= 1) {
        ss += __shfl_xor_sync(0xffffffffu, ss, o);
        if constexpr (BWD) gx += __shfl_xor_sync(0xffffffffu, gx, o);
      }
      const float r = rsqrtf(fmaf(ss, A.inv_d, A.eps));
      const float mean_gu = BWD ? gx * r * A.inv_d : 0.f;
#pragma unroll
      for (int u = 0; u < KU; ++u) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          const float ua = a[u][i] * r, ub = b[u][i] * r;
          if constexpr (BWD) {
            dwa[u][i] = fmaf(ga[u][i], ua, dwa[u][i]);
            dwb[u][i] = fmaf(gb[u][i], ub, dwb[u][i]);
            a[u][i] = r * (ga[u][i] * wa[u][i] - ua * mean_gu);
            b[u][i] = r * (gb[u][i] * wb[u][i] - ub * mean_gu);
          } else {
            const float na = ua * wa[u][i], nb = ub * wb[u][i];
            a[u][i] = fmaf(na, cs[u][i], -nb * sn[u][i]);
            b[u][i] = fmaf(nb, cs[u][i], na * sn[u][i]);
          }
        }
        from_pairs<VEC, INTER>(a[u], b[u]);
        if (live && o1[u] >= 0) store_vec<T, VEC>(ot + o1[u], a[u]);
        if (live && o2[u] >= 0) store_vec<T, VEC>(ot + o2[u], b[u]);
      }
      ot += t.os[1];
    }
  }

  if constexpr (BWD) {
    if (t.dw_part == nullptr) return;  // the same for the whole CTA
#pragma unroll
    for (int u = 0; u < KU; ++u) {
      from_pairs<VEC, INTER>(dwa[u], dwb[u]);
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        if (o1[u] >= 0) sm_dw[grp * D + o1[u] + i] = dwa[u][i];
        if (o2[u] >= 0) sm_dw[grp * D + o2[u] + i] = dwb[u][i];
      }
    }
    __syncthreads();
    float* part = t.dw_part + (static_cast<int64_t>(chunk) * gridDim.x + blockIdx.x) * D;
    for (int d = threadIdx.x; d < D; d += kQkThreads) {
      float s = 0.f;
      for (int g = 0; g < groups; ++g) s += sm_dw[g * D + d];
      part[d] = s;
    }
  }
}

// dw[d] = sum of the partial rows, 32 columns per CTA, 32 row strands added in a fixed order.
__global__ void __launch_bounds__(1024) qk_dw_kernel(const float* p0, const float* p1, int n0, int n1, void* dw0,
                                                     void* dw1, int D, int w_bf16) {
  __shared__ float sm[32][33];
  const float* p = blockIdx.y ? p1 : p0;
  void* dw = blockIdx.y ? dw1 : dw0;
  const int n = blockIdx.y ? n1 : n0;
  if (dw == nullptr) return;
  const int col = blockIdx.x * 32 + threadIdx.x;
  float s = 0.f;
  if (col < D)
#pragma unroll 4
    for (int i = threadIdx.y; i < n; i += 32) s += p[static_cast<int64_t>(i) * D + col];
  sm[threadIdx.y][threadIdx.x] = s;
  __syncthreads();
  if (threadIdx.y == 0 && col < D) {
    s = 0.f;
    for (int i = 0; i < 32; ++i) s += sm[i][threadIdx.x];
    if (w_bf16) static_cast<__nv_bfloat16*>(dw)[col] = __float2bfloat16_rn(s);
    else static_cast<float*>(dw)[col] = s;
  }
}

struct QkPlan {
  int vec, ku, lpr, head_chunk, grid_x, chunks[2];
};

// The widest piece that every offset, stride and base allows; one token per lane group.
QkPlan qk_plan(const trnsparse_qk_norm_rope_args* a, bool bwd) {
  QkPlan p;
  const int es = a->dtype == TRNSPARSE_F32 ? 4 : 2;
  auto fits = [&](int vec) {
    const int bytes = vec * es;
    const uintptr_t bmask = static_cast<uintptr_t>(bytes - 1);
    if (a->rotary_dim % (2 * vec) || (a->head_dim - a->rotary_dim) % (2 * vec)) return false;
    for (int i = 0; i < 2; ++i) {
      if ((reinterpret_cast<uintptr_t>(a->x[i]) | reinterpret_cast<uintptr_t>(a->out[i])) & bmask) return false;
      if (bwd && (reinterpret_cast<uintptr_t>(a->dy[i]) & bmask)) return false;
      for (int j = 0; j < 3; ++j) {
        if (a->x_strides[i][j] % vec || a->out_strides[i][j] % vec) return false;
        if (bwd && a->dy_strides[i][j] % vec) return false;
      }
    }
    return true;
  };
  // four elements a piece for both types: bf16 pieces of eight need twice the registers (148 in the backward pass, one
  // CTA an SM, which took 1.9 times as long at 16384 tokens of 2 x 16 heads of 128)
  p.vec = fits(4) ? 4 : 1;
  const int units = static_cast<int>((a->head_dim + 2 * p.vec - 1) / (2 * p.vec));
  p.lpr = 1;
  while (p.lpr < units && p.lpr < 32) p.lpr *= 2;
  p.ku = p.vec == 1 ? 4 : 1;
  const int groups = kQkThreads / p.lpr;
  const int64_t tgroups = (a->batch * a->seq + groups - 1) / groups;
  // Many heads per group share one set of angles; few tokens want every head on a group of its own.
  const int sms = sm_count();
  p.head_chunk = 16;
  auto blocks = [&](int hc) {
    return tgroups * ((a->heads[0] + hc - 1) / hc + (a->heads[1] + hc - 1) / hc);
  };
  while (p.head_chunk > 1 && blocks(p.head_chunk) < 8 * sms) p.head_chunk /= 2;
  for (int i = 0; i < 2; ++i) p.chunks[i] = static_cast<int>((a->heads[i] + p.head_chunk - 1) / p.head_chunk);
  // Forward: a token group a CTA (up to a bound). Backward: as few CTAs as fill the GPU once, each with the same
  // number of groups, because every CTA leaves a partial row of dw to be added.
  const int chunks = p.chunks[0] + p.chunks[1];
  int64_t cap = bwd ? 2ll * sms / (chunks > 0 ? chunks : 1) : 64ll * sms;
  if (cap < 1) cap = 1;
  const int64_t each = (tgroups + cap - 1) / cap;
  p.grid_x = static_cast<int>((tgroups + each - 1) / each);
  return p;
}

template <typename T, int VEC, int KU, bool INTER, bool BWD>
int qk_launch(const QkArgs& A, const QkPlan& p, cudaStream_t st) {
  // 256 / lpr groups of D floats: 8 KB at most over all plans (head_dim 256 on 32 lanes, 8 on one)
  const size_t smem = BWD ? sizeof(float) * static_cast<size_t>(kQkThreads / p.lpr) * A.D : 0;
  auto kern = qk_norm_rope_kernel<T, VEC, KU, INTER, BWD>;
  kern<<<dim3(p.grid_x, p.chunks[0] + p.chunks[1]), kQkThreads, smem, st>>>(A, p.lpr);
  TSB_CHECK_LAUNCH("qk_norm_rope launch");
  return TRNSPARSE_OK;
}

template <bool INTER, bool BWD>
int qk_dispatch(const QkArgs& A, const QkPlan& p, bool f32, cudaStream_t st) {
  if (f32) {
    if (p.vec == 4) return qk_launch<float, 4, 1, INTER, BWD>(A, p, st);
    return qk_launch<float, 1, 4, INTER, BWD>(A, p, st);
  }
  if (p.vec == 4) return qk_launch<__nv_bfloat16, 4, 1, INTER, BWD>(A, p, st);
  return qk_launch<__nv_bfloat16, 1, 4, INTER, BWD>(A, p, st);
}

int qk_check(const trnsparse_qk_norm_rope_args* a) {
  TSB_REQUIRE(a != nullptr, "qk_norm_rope: null arguments");
  TSB_REQUIRE(a->batch >= 0 && a->batch < (1ll << 31) && a->seq >= 0 && a->seq < (1ll << 31) && a->heads[0] >= 0 && a->heads[1] >= 0 &&
                  a->heads[0] < 32768 && a->heads[1] < 32768,
              "qk_norm_rope: bad sizes");
  TSB_REQUIRE(a->head_dim >= 1 && a->head_dim <= 256, "qk_norm_rope: head_dim must be in [1, 256] (got %lld)",
              (long long)a->head_dim);
  TSB_REQUIRE(a->rotary_dim >= 0 && a->rotary_dim % 2 == 0 && a->rotary_dim <= a->head_dim,
              "qk_norm_rope: rotary_dim must be even and at most head_dim (got %lld)", (long long)a->rotary_dim);
  if (a->dtype != TRNSPARSE_F32 && a->dtype != TRNSPARSE_BF16)
    return fail(TRNSPARSE_ERR_DTYPE, "qk_norm_rope: dtype %d not supported (F32, BF16)", a->dtype);
  if (a->weight_dtype != TRNSPARSE_F32 && a->weight_dtype != TRNSPARSE_BF16)
    return fail(TRNSPARSE_ERR_DTYPE, "qk_norm_rope: weight dtype %d not supported (F32, BF16)", a->weight_dtype);
  if (a->position_type != TRNSPARSE_I32 && a->position_type != TRNSPARSE_I64)
    return fail(TRNSPARSE_ERR_DTYPE, "qk_norm_rope: position type %d not supported (I32, I64)", a->position_type);
  return TRNSPARSE_OK;
}

int qk_run(const trnsparse_qk_norm_rope_args* a, bool bwd, void* ws, size_t ws_bytes, void* stream) {
  int rc = qk_check(a);
  if (rc) return rc;
  cudaStream_t st = as_stream(stream);
  const bool empty = a->batch == 0 || a->seq == 0 || (a->heads[0] == 0 && a->heads[1] == 0);
  const int wes = a->weight_dtype == TRNSPARSE_F32 ? 4 : 2;
  if (empty) {
    for (int i = 0; bwd && i < 2; ++i)
      if (a->dw[i]) {
        cudaError_t e = cudaMemsetAsync(a->dw[i], 0, static_cast<size_t>(wes * a->head_dim), st);
        if (e != cudaSuccess) return cuda_status(e, "qk_norm_rope: zero dw");
      }
    return TRNSPARSE_OK;
  }
  TSB_REQUIRE(a->positions && (a->rotary_dim == 0 || a->inv_freq), "qk_norm_rope: null pointer");
  QkArgs A = {};
  const QkPlan p = qk_plan(a, bwd);
  float* part = static_cast<float*>(ws);
  if (bwd) TSB_REQUIRE(ws && ws_bytes >= trnsparse_qk_norm_rope_workspace_size(a), "qk_norm_rope: workspace too small");
  for (int i = 0; i < 2; ++i) {
    QkTensor& t = A.t[i];
    TSB_REQUIRE(a->heads[i] == 0 || (a->x[i] && a->out[i] && (!bwd || a->dy[i])), "qk_norm_rope: null pointer");
    t.x = a->x[i];
    t.dy = a->dy[i];
    t.out = a->out[i];
    t.w = a->weight[i];
    for (int j = 0; j < 3; ++j) {
      t.xs[j] = a->x_strides[i][j];
      t.dys[j] = a->dy_strides[i][j];
      t.os[j] = a->out_strides[i][j];
    }
    t.heads = static_cast<int>(a->heads[i]);
    t.chunks = p.chunks[i];
    if (bwd && a->dw[i]) t.dw_part = part;
    part += static_cast<int64_t>(p.chunks[i]) * p.grid_x * a->head_dim;
  }
  A.pos = a->positions;
  A.freq = a->inv_freq;
  A.tokens = a->batch * a->seq;
  A.pos_stride = a->position_batch_stride;
  A.S = static_cast<int>(a->seq);
  A.D = static_cast<int>(a->head_dim);
  A.R = static_cast<int>(a->rotary_dim);
  A.pos64 = a->position_type == TRNSPARSE_I64;
  A.w_bf16 = a->weight_dtype == TRNSPARSE_BF16;
  A.head_chunk = p.head_chunk;
  A.eps = static_cast<float>(a->eps);
  A.inv_d = 1.f / static_cast<float>(a->head_dim);
  const bool f32 = a->dtype == TRNSPARSE_F32;
  if (bwd) rc = a->interleaved ? qk_dispatch<true, true>(A, p, f32, st) : qk_dispatch<false, true>(A, p, f32, st);
  else rc = a->interleaved ? qk_dispatch<true, false>(A, p, f32, st) : qk_dispatch<false, false>(A, p, f32, st);
  if (rc || !bwd || (!a->dw[0] && !a->dw[1])) return rc;
  const int n0 = p.chunks[0] * p.grid_x, n1 = p.chunks[1] * p.grid_x;
  qk_dw_kernel<<<dim3((A.D + 31) / 32, 2), dim3(32, 32), 0, st>>>(A.t[0].dw_part, A.t[1].dw_part, n0, n1, a->dw[0],
                                                                  a->dw[1], A.D, A.w_bf16);
  TSB_CHECK_LAUNCH("qk_norm_rope dw launch");
  return TRNSPARSE_OK;
}

}  // namespace
}  // namespace tsb

using namespace tsb;

extern "C" int trnsparse_qk_norm_rope(const trnsparse_qk_norm_rope_args* args, void* stream) {
  return qk_run(args, false, nullptr, 0, stream);
}

extern "C" size_t trnsparse_qk_norm_rope_workspace_size(const trnsparse_qk_norm_rope_args* args) {
  if (qk_check(args) != TRNSPARSE_OK || args->batch * args->seq == 0) return 0;
  const QkPlan p = qk_plan(args, true);
  return sizeof(float) * static_cast<size_t>(p.chunks[0] + p.chunks[1]) * p.grid_x * args->head_dim;
}

extern "C" int trnsparse_qk_norm_rope_backward(const trnsparse_qk_norm_rope_args* args, void* ws, size_t ws_bytes,
                                               void* stream) {
  return qk_run(args, true, ws, ws_bytes, stream);
}
